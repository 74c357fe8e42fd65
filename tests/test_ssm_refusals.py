"""Refusals of the selective state space operators and of qk_norm_rope, without a GPU: the Python
checks (shapes, types, CPU tensors), and the C entry points' own, before any HIP call."""

import ctypes
import os
import re
import struct

import pytest
import torch

from tops import _lib
from tops.ops.rope import qk_norm_rope, rotary_inv_freq
from tops.ops.ssm import (causal_conv1d, causal_conv1d_step, selective_scan, selective_scan_step)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def z(*s, dt=torch.float32):
    return torch.zeros(*s, dtype=dt)


def scan_args(**over):
    a = dict(u=z(2, 4, 6), delta=z(2, 4, 6), A=z(6, 3), B=z(2, 4, 3), C=z(2, 4, 3))
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(u=z(2, 6)), dict(delta=z(2, 4, 5)), dict(z=z(2, 4, 7)), dict(A=z(5, 3)), dict(A=z(6)),
    dict(A=z(6, 65), B=z(2, 4, 65), C=z(2, 4, 65)), dict(A=z(6, 0), B=z(2, 4, 0), C=z(2, 4, 0)),
    dict(B=z(2, 4, 4)), dict(B=z(2, 3, 3)), dict(C=z(2, 4, 1, 3)), dict(B=z(2, 4, 4, 3), C=z(2, 4, 4, 3)),
    dict(B=z(2, 4, 0, 3), C=z(2, 4, 0, 3)), dict(D=z(5)), dict(delta_bias=z(6, 1)),
    dict(initial_state=z(1, 6, 3)), dict(initial_state=z(2, 3, 6)), dict(cu_seqlens=[0, 4]),
])
def test_scan_shapes(over):
    with pytest.raises(ValueError):
        selective_scan(**scan_args(**over))


@pytest.mark.parametrize("cu", [[0], [0, 3], [0, 5], [1, 4], [0, 3, 2, 4], [-1, 4]])
def test_offsets(cu):
    a = {n: t[:1] if t.dim() == 3 else t for n, t in scan_args().items()}
    with pytest.raises(ValueError, match="cu_seqlens"):
        selective_scan(**a, cu_seqlens=cu)
    with pytest.raises(ValueError, match="cu_seqlens"):
        causal_conv1d(z(1, 4, 6), z(6, 4), cu_seqlens=cu)


def test_no_cpu_path():
    for f in (lambda: selective_scan(**scan_args()),
              lambda: selective_scan(**scan_args(u=z(2, 4, 6).requires_grad_())),
              lambda: selective_scan_step(z(2, 6, 3), z(2, 6), z(2, 6), z(6, 3), z(2, 3), z(2, 3)),
              lambda: causal_conv1d(z(2, 4, 6), z(6, 4)),
              lambda: causal_conv1d_step(z(2, 6), z(2, 4, 6), z(6, 4)),
              lambda: qk_norm_rope(z(1, 2, 3, 8), z(1, 2, 1, 8))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            f()


def step_args(**over):
    a = dict(state=z(2, 6, 3), u=z(2, 6), delta=z(2, 6), A=z(6, 3), B=z(2, 3), C=z(2, 3))
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(state=z(1, 6, 3)), dict(state=z(2, 3, 6)), dict(state=z(2, 6, 3, dt=torch.bfloat16)),
    dict(state=z(2, 3, 6).transpose(1, 2)), dict(u=z(2, 1, 6)), dict(delta=z(2, 5)),
    dict(z=z(1, 6)), dict(B=z(2, 4)), dict(C=z(1, 3)), dict(B=z(2, 4, 3), C=z(2, 4, 3)),
    dict(D=z(5)), dict(delta_bias=z(3)), dict(state_indices=z(3, dt=torch.int32)),
    dict(state_indices=z(2)), dict(state_indices=z(4, dt=torch.int64)[::2]),
])
def test_scan_step_shapes(over):
    with pytest.raises(ValueError):
        selective_scan_step(**step_args(**over))


def test_steps_have_no_gradient():
    with pytest.raises(RuntimeError, match="no_grad"):
        selective_scan_step(**step_args(A=z(6, 3).requires_grad_()))
    with pytest.raises(RuntimeError, match="no_grad"):
        causal_conv1d_step(z(2, 6), z(2, 4, 6), z(6, 4).requires_grad_())


@pytest.mark.parametrize("over", [
    dict(x=z(2, 6)), dict(weight=z(5, 4)), dict(weight=z(6, 9)), dict(weight=z(6, 0)),
    dict(weight=z(6, 2, 4)), dict(bias=z(5)), dict(activation="gelu"),
    dict(initial_state=z(2, 3, 6)), dict(initial_state=z(1, 4, 6)), dict(cu_seqlens=[0, 4])])
def test_conv_shapes(over):
    a = dict(x=z(2, 4, 6), weight=z(6, 4))
    a.update(over)
    with pytest.raises(ValueError):
        causal_conv1d(**a)


@pytest.mark.parametrize("over", [
    dict(x=z(2, 1, 6)), dict(weight=z(6, 9)), dict(state=z(2, 3, 6)), dict(state=z(1, 4, 6)),
    dict(state=z(2, 4, 6, dt=torch.bfloat16)), dict(state=z(2, 6, 4).transpose(1, 2)),
    dict(bias=z(4)), dict(activation="relu"), dict(state_indices=z(1, dt=torch.int64))])
def test_conv_step_shapes(over):
    a = dict(x=z(2, 6), state=z(2, 4, 6), weight=z(6, 4))
    a.update(over)
    with pytest.raises(ValueError):
        causal_conv1d_step(**a)


def test_conv_step_types():
    with pytest.raises((TypeError, RuntimeError)):
        causal_conv1d_step(z(2, 6, dt=torch.float16), z(2, 4, 6, dt=torch.float16), z(6, 4))


@pytest.mark.parametrize("over", [
    dict(q=z(2, 3, 8)), dict(k=z(1, 3, 1, 8)), dict(k=z(2, 3, 1, 6)),
    dict(q=z(2, 3, 1, 513), k=z(2, 3, 1, 513)), dict(q_weight=z(7)), dict(k_weight=z(1, 8)),
    dict(inv_freq=z(4)), dict(inv_freq=z(5, dt=torch.float64)),
    dict(inv_freq=z(2, 2, dt=torch.float64)), dict(positions=z(2, 3)),
    dict(positions=z(2, dt=torch.int64)), dict(positions=z(1, 3, dt=torch.int64))])
def test_qk_shapes(over):
    a = dict(q=z(2, 3, 4, 8), k=z(2, 3, 1, 8))
    a.update(over)
    with pytest.raises(ValueError):
        qk_norm_rope(**a)


def test_odd_rotary_dim():
    with pytest.raises(ValueError):
        rotary_inv_freq(7)


# ---------------------------------------------------------------------------
# the C entry points
# ---------------------------------------------------------------------------


def _structs():
    """Field names of every struct of the header, all of them 8 bytes."""
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "tops_gla_ssm.h")).read(),
                 flags=re.S)
    out = {}
    for m in re.finditer(r"typedef struct (\w+) \{(.*?)\}", src, re.S):
        names = []
        for decl in m.group(2).split(";"):
            kind = decl.split()
            if not kind:
                continue
            assert "*" in decl or kind[0] in ("int64_t", "double"), decl
            names += [re.findall(r"\w+", part)[-1] for part in decl.split(",")]
        out[m.group(1)] = names
    return out


STRUCTS = _structs()


def entry(name, struct_name, **fields):
    names = STRUCTS[struct_name]
    assert set(fields) <= set(names), set(fields) - set(names)
    b = b"".join(struct.pack("=d" if isinstance(fields.get(n), float) else "=q", fields.get(n, 0))
                 for n in names)
    lib = _lib.load()
    return getattr(lib, name)(b, None), lib.tops_gla_last_error().decode()


def test_binding_matches_the_header():
    import importlib

    mods = {n: importlib.import_module("tops.ops." + n)
            for n in ("ssm.scan", "ssm.conv", "rope.qk_norm_rope")}
    for s, size in (("tops_gla_scan_args", mods["ssm.scan"]._ARGS.size),
                    ("tops_gla_scan_step_args", mods["ssm.scan"]._STEP.size),
                    ("tops_gla_conv_args", mods["ssm.conv"]._ARGS.size),
                    ("tops_gla_conv_step_args", mods["ssm.conv"]._STEP.size),
                    ("tops_gla_qk_args", mods["rope.qk_norm_rope"]._ARGS.size)):
        assert size == 8 * len(STRUCTS[s]), s
    src = open(os.path.join(ROOT, "include", "tops_gla_ssm.h")).read()
    assert set(re.findall(r"\b(?:int|int64_t) (tops_gla_\w+)\(", src)) == set(_lib._SSM_SIGS)


SCAN = dict(batch=1, nseq=1, T=4, D=8, N=4, G=1, piece=64, dtype=1)


@pytest.mark.parametrize("over,code,what", [
    (dict(dtype=7), 1, "dtype"), (dict(N=65), 2, "N must"), (dict(N=0), 2, "N must"),
    (dict(D=0), 1, "D must"), (dict(G=3), 1, "divide"), (dict(G=0), 1, "divide"),
    (dict(piece=24), 1, "piece"), (dict(piece=0), 1, "piece"), (dict(T=-1), 1, "bad"),
    (dict(batch=1 << 20, nseq=1 << 20, T=1 << 20), 2, "2^31"), (dict(nseq=2), 1, "nseq"),
    (dict(segs=64, batch=2), 1, "batch == 1"), (dict(segs=64, nsegs=0), 1, "nsegs"),
    (dict(T=65), 1, "piece_h"), (dict(segs=64, nsegs=2, piece_h=64), 1, "piece_dt"),
    (dict(), 1, "NULL"), (dict(A=64, u=64, delta=64, B=64, C=64), 1, "y must"),
])
def test_scan_entry(over, code, what):
    rc, msg = entry("tops_gla_selective_scan_fwd", "tops_gla_scan_args", **{**SCAN, **over})
    assert rc == code and what in msg, msg


@pytest.mark.parametrize("over,what", [
    (dict(), "chunk_h"), (dict(chunk_h=64, z=64), "dz"), (dict(chunk_h=64), "dA"),
    (dict(chunk_h=64, dA=64), "ws"), (dict(chunk_h=64, dA=64, ws=64, ws_bytes=64), "ws")])
def test_scan_bwd_entry(over, what):
    a = {**SCAN, **dict.fromkeys(("A", "u", "delta", "B", "C"), 64)}
    if over:
        a.update(dict.fromkeys(("dy", "du", "ddelta", "dB", "dC"), 64))
    rc, msg = entry("tops_gla_selective_scan_bwd", "tops_gla_scan_args", **{**a, **over})
    assert rc == 1 and what in msg, msg


def test_step_entries():
    s = dict(batch=2, slots=1, D=8, N=4, G=1, W=4, dtype=1)
    scan = {k: v for k, v in s.items() if k != "W"}
    conv = {k: v for k, v in s.items() if k not in ("N", "G")}
    rc, msg = entry("tops_gla_selective_scan_step", "tops_gla_scan_step_args", **scan)
    assert rc == 1 and "batch" in msg
    rc, msg = entry("tops_gla_selective_scan_step", "tops_gla_scan_step_args", **{**scan, "slots": 2})
    assert rc == 1 and "NULL" in msg
    rc, msg = entry("tops_gla_causal_conv_step", "tops_gla_conv_step_args", **conv)
    assert rc == 1 and "batch" in msg
    rc, msg = entry("tops_gla_causal_conv_step", "tops_gla_conv_step_args", **{**conv, "W": 9})
    assert rc == 2 and "W in 1..8" in msg
    rc, msg = entry("tops_gla_causal_conv_step", "tops_gla_conv_step_args",
                    **{**conv, "w_dtype": 2})
    assert rc == 1 and "dtype" in msg


@pytest.mark.parametrize("over,code,what", [
    (dict(dtype=2), 1, "dtype"), (dict(W=0), 2, "W in"), (dict(D=0), 1, "D must"),
    (dict(nseq=3), 1, "nseq"), (dict(cu=64, batch=2), 1, "batch == 1"), (dict(T=-2), 1, "bad"),
    (dict(), 1, "w must"), (dict(w=64), 1, "x must"), (dict(w=64, x=64), 1, "y must")])
def test_conv_entry(over, code, what):
    rc, msg = entry("tops_gla_causal_conv_fwd", "tops_gla_conv_args",
                    **{**dict(batch=1, nseq=1, T=4, D=8, W=4, dtype=0), **over})
    assert rc == code and what in msg, msg


def test_conv_bwd_entry():
    a = dict(batch=1, nseq=1, T=4, D=8, W=4, dtype=0, x=64, w=64)
    rc, msg = entry("tops_gla_causal_conv_bwd", "tops_gla_conv_args", **a)
    assert rc == 1 and "dy" in msg
    rc, msg = entry("tops_gla_causal_conv_bwd", "tops_gla_conv_args",
                    **{**a, "dy": 64, "dx": 64, "dw": 64, "dbias": 64})
    assert rc == 1 and "ws" in msg


@pytest.mark.parametrize("over,code,what", [
    (dict(dtype=5), 1, "dtype"), (dict(D=513), 2, "D must"), (dict(R=3), 1, "R must"),
    (dict(R=18), 1, "R must"), (dict(R=4), 1, "inv_freq"), (dict(Hq=-1), 1, "bad"), (dict(), 1, "NULL")])
def test_qk_entry(over, code, what):
    rc, msg = entry("tops_gla_qk_norm_rope_fwd", "tops_gla_qk_args",
                    **{**dict(batch=1, T=2, Hq=2, Hk=1, D=16, dtype=1, eps=1e-6), **over})
    assert rc == code and what in msg, msg


def test_null_arguments():
    lib = _lib.load()
    for name, sig in _lib._SSM_SIGS.items():
        if sig[0] is ctypes.c_char_p:
            assert getattr(lib, name)(None, None) == 1
            assert b"NULL" in lib.tops_gla_last_error()


@pytest.mark.parametrize("T,fits", [((1 << 31) - 64, True), ((1 << 31) - 63, False),
                                    ((1 << 31) - 1, False)])
def test_scan_entry_tokens(T, fits):
    """The kernels' token indices go up to a tile past the last token, in 32 bits."""
    rc, msg = entry("tops_gla_selective_scan_fwd", "tops_gla_scan_args",
                    **{**SCAN, "T": T, "D": 1, "N": 1, "piece": 1 << 22, "piece_h": 64,
                       "piece_dt": 64})
    assert (rc, ("A must" if fits else "2^31") in msg) == (1 if fits else 2, True), msg


@pytest.mark.parametrize("state", [
    z(1, 6, 3).expand(2, 6, 3), z(100).as_strided((2, 6, 3), (17, 3, 1)),
    z(100).as_strided((3, 6, 3), (9, 3, 1))])
def test_scan_step_slots_that_overlap(state):
    with pytest.raises(ValueError, match="slots"):
        selective_scan_step(**step_args(state=state))


@pytest.mark.parametrize("state", [
    z(1, 4, 6).expand(2, 4, 6), z(100).as_strided((2, 4, 6), (23, 6, 1))])
def test_conv_step_slots_that_overlap(state):
    with pytest.raises(ValueError, match="slots"):
        causal_conv1d_step(z(2, 6), state, z(6, 4))


@pytest.mark.parametrize("state", [z(100).as_strided((1, 6, 3), (0, 3, 1)),
                                   z(100).as_strided((2, 6, 3), (18, 3, 1)),
                                   z(100).as_strided((2, 6, 3), (20, 3, 1))])
def test_scan_step_slots_that_do_not(state):
    a = step_args(state=state)
    n = state.shape[0]
    a.update({k: a[k][:n] for k in ("u", "delta", "B", "C")})
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        selective_scan_step(**a)


def test_step_entries_with_slots_that_overlap():
    ptrs = dict.fromkeys(("state", "u", "delta", "B", "C", "A", "y", "x", "w"), 64)
    scan = dict(batch=2, slots=2, D=8, N=4, G=1, dtype=1, state_ss=31)
    conv = dict(batch=2, slots=2, D=8, W=4, dtype=1, state_ss=31)
    for name, s, a in (("tops_gla_selective_scan_step", "tops_gla_scan_step_args", scan),
                       ("tops_gla_causal_conv_step", "tops_gla_conv_step_args", conv)):
        rc, msg = entry(name, s, **{**a, **{k: v for k, v in ptrs.items() if k in STRUCTS[s]}})
        assert rc == 1 and "overlap" in msg, msg


@pytest.mark.parametrize("T", [64, 65, 1 << 20])
def test_scan_entry_of_an_empty_batch(T):
    """No sequences: one piece each, whatever their length, and nothing to launch for them."""
    lib = _lib.load()
    piece = lib.tops_gla_selective_scan_piece(0, 0, 8, 4, 1)
    rc, msg = entry("tops_gla_selective_scan_fwd", "tops_gla_scan_args",
                    **{**SCAN, "batch": 0, "nseq": 0, "T": T, "piece": piece})
    assert rc == 1 and "A must" in msg, msg   # the check after those of the pieces
    rc, msg = entry("tops_gla_selective_scan_fwd", "tops_gla_scan_args",
                    **{**SCAN, "batch": 0, "nseq": 0, "T": T, "piece": piece, "A": 64})
    assert rc == 1 and "bc must" in msg, msg


def test_tables_of_two_threads(monkeypatch):
    """A table made by one thread while another looks one up in a capture."""
    import importlib
    import threading

    common = importlib.import_module("tops.ops.ssm._common")
    second, tensor = [], torch.tensor

    class Tables(dict):
        def items(self):
            it = iter(super().items())
            yield next(it)
            second.append(threading.Thread(target=make, args=("b",)))
            second[0].start()
            second[0].join(0.2)
            yield from it

    def make(key):
        return common.device_table(key, lambda: ([1], key), torch.device("cpu"))

    monkeypatch.setattr(common, "_tables", Tables())
    monkeypatch.setattr(common, "_held", [])
    monkeypatch.setattr(common, "stream_of", lambda d: ctypes.c_void_p(streams.pop(0)))
    monkeypatch.setattr(torch, "tensor", lambda v, dtype, pin_memory: tensor(v, dtype=dtype))
    capturing = threading.local()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing",
                        lambda: getattr(capturing, "now", False))
    streams = [1, 1, 2, 1]
    make("x")
    want = make("a")
    capturing.now = True   # stream 2, whose own table it cannot make
    assert make("a") is want
    second[0].join()
    assert len(common._tables) == 3
