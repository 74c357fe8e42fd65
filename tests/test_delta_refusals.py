"""Refusals of the gated delta rule and of the layer norm, without a GPU: the Python checks (shapes,
types, CPU tensors), and the C entry points' own, before any HIP call. And the oracle against
differences."""

import ctypes
import importlib
import os
import re
import struct

import pytest
import torch

from delta_ref import F64, delta, layer_norm as ref_norm
from tops import _lib
from tops.modules import LayerNorm
from tops.ops.delta import gated_delta_rule, gated_delta_rule_step
from tops.ops.norm import layer_norm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def z(*s, dt=torch.float32):
    return torch.zeros(*s, dtype=dt)


def args(**over):
    a = dict(q=z(2, 4, 2, 8), k=z(2, 4, 2, 8), v=z(2, 4, 4, 16), g=z(2, 4, 4), beta=z(2, 4, 4))
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(q=z(2, 4, 8)), dict(k=z(2, 4, 2, 9)), dict(k=z(2, 4, 1, 8)), dict(v=z(2, 4, 16)),
    dict(v=z(2, 5, 4, 16)), dict(v=z(2, 4, 3, 16), g=z(2, 4, 3), beta=z(2, 4, 3)),
    dict(v=z(2, 4, 4, 0)), dict(q=z(2, 4, 2, 0), k=z(2, 4, 2, 0)), dict(g=z(2, 4, 2)),
    dict(beta=z(2, 4)), dict(g=z(2, 4, 4, 1)), dict(initial_state=z(2, 4, 16, 8)),
    dict(initial_state=z(1, 4, 8, 16)), dict(cu_seqlens=[0, 4]),
    dict(q=z(2, 4, 0, 8), k=z(2, 4, 0, 8))])
def test_shapes(over):
    with pytest.raises(ValueError):
        gated_delta_rule(**args(**over))


def test_wide_keys():
    a = args(q=z(2, 4, 2, 257), k=z(2, 4, 2, 257))
    with pytest.raises(NotImplementedError, match="256"):
        gated_delta_rule(**a)
    with pytest.raises(NotImplementedError, match="256"):
        gated_delta_rule_step(z(2, 4, 257, 16), **a)


@pytest.mark.parametrize("cu", [[0], [0, 3], [0, 5], [1, 4], [0, 3, 2, 4], [-1, 4]])
def test_offsets(cu):
    with pytest.raises(ValueError, match="cu_seqlens"):
        gated_delta_rule(**{n: t[:1] for n, t in args().items()}, cu_seqlens=cu)


def step_args(**over):
    a = dict(state=z(2, 4, 8, 16), **{n: t[:, 0] for n, t in args().items()})
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(state=z(1, 4, 8, 16)), dict(state=z(2, 4, 16, 8)),
    dict(state=z(2, 4, 8, 16, dt=torch.bfloat16)), dict(state=z(2, 4, 16, 8).transpose(2, 3)),
    dict(state=z(2, 8, 4, 16).transpose(1, 2)), dict(state=z(1, 4, 8, 16).expand(2, 4, 8, 16)),
    dict(state=z(2000).as_strided((2, 4, 8, 16), (511, 128, 16, 1))), dict(q=z(2, 8)),
    dict(k=z(2, 2, 9)), dict(v=z(1, 4, 16)), dict(v=z(2, 1, 4, 16)), dict(g=z(2, 2)),
    dict(beta=z(2, 1, 4)), dict(state_indices=z(3, dt=torch.int32)), dict(state_indices=z(2)),
    dict(state_indices=z(4, dt=torch.int64)[::2])])
def test_step_shapes(over):
    with pytest.raises(ValueError):
        gated_delta_rule_step(**step_args(**over))


def test_steps_have_no_gradient():
    with pytest.raises(RuntimeError, match="no_grad"):
        gated_delta_rule_step(**step_args(g=z(2, 4).requires_grad_()))


@pytest.mark.parametrize("over", [
    dict(x=z(())), dict(x=z(3, 0)), dict(weight=z(5)), dict(weight=z(1, 6)), dict(bias=z(7)),
    dict(eps=-1e-5), dict(eps=float("nan"))])
def test_norm_arguments(over):
    a = dict(x=z(3, 6), weight=z(6), bias=z(6))
    a.update(over)
    with pytest.raises(ValueError):
        layer_norm(**a)


def test_no_cpu_path():
    for f in (lambda: gated_delta_rule(**args()),
              lambda: gated_delta_rule(**args(q=z(2, 4, 2, 8).requires_grad_())),
              lambda: gated_delta_rule(**args(q=z(2, 4, 2, 3), k=z(2, 4, 2, 3))),
              lambda: gated_delta_rule_step(**step_args()),
              lambda: layer_norm(z(3, 6)), lambda: LayerNorm(6)(z(3, 6))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            f()


# ---------------------------------------------------------------------------
# the C entry points
# ---------------------------------------------------------------------------


def structs():
    """Fields of the header's structs, in order: {struct: [(name, is a double)]}."""
    src = open(os.path.join(ROOT, "include", "tops_gla_delta.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    out = {}
    for body, name in re.findall(r"typedef struct \w+ \{(.*?)\} (\w+);", src, flags=re.S):
        out[name] = [(re.sub(r"[*\s]", "", f), kind == "double")
                     for kind, fs in re.findall(r"(?:const )?(\w+) ([^;]+);", body)
                     for f in fs.split(",")]
    return out


STRUCTS = structs()


def entry(name, s, **fields):
    assert set(fields) <= {f for f, _ in STRUCTS[s]}, set(fields) - {f for f, _ in STRUCTS[s]}
    raw = b"".join(struct.pack("=d" if d else "=q", fields.get(f, 0)) for f, d in STRUCTS[s])
    rc = getattr(_lib.load(), name)(raw, None)
    return rc, _lib.load().tops_gla_last_error().decode()


def test_binding_matches_the_header():
    import importlib

    dmod = importlib.import_module("tops.ops.delta.gated_delta_rule")
    nmod = importlib.import_module("tops.ops.norm.layer_norm")
    for s, packed in (("tops_gla_delta_args", dmod._ARGS), ("tops_gla_delta_step_args", dmod._STEP),
                      ("tops_gla_layer_norm_args", nmod._ARGS)):
        kinds = "".join("d" if d else "q" for _, d in STRUCTS[s])
        spelt = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", packed.format))
        assert kinds == spelt, s
    src = open(os.path.join(ROOT, "include", "tops_gla_delta.h")).read()
    assert set(re.findall(r"\b(?:int|int64_t) (tops_gla_\w+)\(", src)) == set(_lib._DELTA_SIGS)


DELTA = dict(batch=1, nseq=1, T=4, H=1, HV=2, K=16, V=16, chunks=1, nsegs=1, seg_chunks=4,
             dtype=1)
PTRS = dict.fromkeys(("q", "k", "v", "g", "beta", "o"), 64)


@pytest.mark.parametrize("over,code,what", [
    (dict(dtype=7), 1, "dtype"), (dict(g_dtype=2), 1, "dtype"), (dict(beta_dtype=-1), 1, "dtype"),
    (dict(K=0), 2, "K must"), (dict(K=257), 2, "K must"), (dict(K=7), 2, "at least 8"),
    (dict(V=4), 2, "at least 8"), (dict(V=0), 2, "V must"), (dict(V=65537), 2, "V must"),
    (dict(H=0), 1, "divide"), (dict(HV=3, H=2), 1, "divide"), (dict(T=-1), 1, "bad"),
    (dict(chunks=2), 1, "chunks"), (dict(nseq=2), 1, "nseq"), (dict(T=65), 1, "chunks"), (dict(nsegs=2), 1, "nsegs"),
    (dict(seg_chunks=0), 1, "seg_chunks"), (dict(seg_chunks=1 << 26), 1, "seg_chunks"),
    (dict(T=320, chunks=5), 1, "nsegs"), (dict(seqs=64, nsegs=0), 1, "bad nseq"),
    (dict(seqs=64, nsegs=3), 1, "bad nseq"),
    (dict(T=65, dtype=0, chunks=2), 1, "chunks"), (dict(seqs=64, batch=2), 1, "batch == 1"),
    (dict(seqs=64, chunks=3), 1, "bad nseq, chunks"), (dict(seqs=64, chunks=0), 1, "bad nseq"),
    (dict(batch=1 << 20, nseq=1 << 20, T=1 << 20), 2, "2^31"),
    (dict(PTRS, q_st=1 << 24), 2, "2^24"), (dict(PTRS, v_st=-1), 2, "2^24"), (dict(PTRS, HV=1 << 10, V=1 << 14), 2, "2^24"),
    (dict(T=(1 << 31) - 64, chunks=(1 << 25) - 1), 2, "2^31"),
    (dict(T=1 << 30, chunks=1 << 24, nsegs=1 << 22, HV=1 << 12), 2, "grid"), (dict(), 1, "NULL"),
    (dict(PTRS, o=0), 1, "o must"), (PTRS, 1, "keep"), (dict(PTRS, keep=256), 1, "keep"),
    (dict(PTRS, keep=128, keep_bytes=1 << 30), 1, "keep")])
def test_delta_entry(over, code, what):
    rc, msg = entry("tops_gla_delta_fwd", "tops_gla_delta_args", **{**DELTA, **over})
    assert rc == code and what in msg, msg


@pytest.mark.parametrize("over,what", [
    (dict(), "dout"), (dict.fromkeys(("dout", "dq", "dk", "dv", "dg"), 64), "dbeta"),
    (dict.fromkeys(("dout", "dq", "dk", "dv", "dg", "dbeta"), 64), "ws"),
    (dict(dict.fromkeys(("dout", "dq", "dk", "dv", "dg", "dbeta"), 64), ws=256, ws_bytes=100),
     "ws")])
def test_delta_bwd_entry(over, what):
    rc, msg = entry("tops_gla_delta_bwd", "tops_gla_delta_args",
                    **{**DELTA, **PTRS, "keep": 256, "keep_bytes": 1 << 30, **over})
    assert rc == 1 and what in msg, msg


STEP = dict(batch=2, slots=2, T=1, H=1, HV=2, K=8, V=4, dtype=1, state_ss=64)


@pytest.mark.parametrize("over,code,what", [
    (dict(dtype=3), 1, "dtype"), (dict(K=300), 2, "K must"), (dict(V=0), 2, "V must"),
    (dict(H=3), 1, "divide"), (dict(slots=1), 1, "batch"), (dict(T=-1), 1, "bad"),
    (dict(), 1, "NULL"), (PTRS, 1, "state must"), (dict(PTRS, state=64, state_ss=63), 1, "overlap"),
    (dict(batch=1 << 30, slots=1 << 30), 2, "grid")])
def test_step_entry(over, code, what):
    rc, msg = entry("tops_gla_delta_step", "tops_gla_delta_step_args", **{**STEP, **over})
    assert rc == code and what in msg, msg


@pytest.mark.parametrize("over,code,what", [
    (dict(dtype=2), 1, "dtype"), (dict(D=0), 2, "D must"), (dict(D=16385), 2, "D must"),
    (dict(rows=-1), 1, "rows"), (dict(), 1, "x must"), (dict(x=64), 1, "y must")])
def test_norm_entry(over, code, what):
    rc, msg = entry("tops_gla_layer_norm_fwd", "tops_gla_layer_norm_args",
                    **{**dict(rows=2, D=8, x_st=8), **over})
    assert rc == code and what in msg, msg


@pytest.mark.parametrize("over,what", [
    (dict(), "stats"), (dict(stats=64, dy=64, dx=64, dw=64), "ws"),
    (dict(stats=64, dy=64, dx=64, db=64, ws=64, ws_bytes=8), "ws")])
def test_norm_bwd_entry(over, what):
    rc, msg = entry("tops_gla_layer_norm_bwd", "tops_gla_layer_norm_args",
                    **{**dict(rows=2, D=8, x_st=8, x=64), **over})
    assert rc == 1 and what in msg, msg


def test_null_arguments():
    lib = _lib.load()
    for name, sig in _lib._DELTA_SIGS.items():
        if sig == [ctypes.c_char_p, ctypes.c_void_p]:
            assert getattr(lib, name)(None, None) == 1
            assert b"NULL" in lib.tops_gla_last_error()


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.tops_gla_layer_norm_ws_bytes(0, 8, 0) == 64
    assert lib.tops_gla_layer_norm_ws_bytes(5, 0, 0) == 0
    assert lib.tops_gla_delta_chunk(1) == 64 and lib.tops_gla_delta_chunk(0) == 32
    assert lib.tops_gla_delta_chunk(2) == 0

    def size(back, nseq=1, chunks=3, nsegs=1, HV=2, K=100, V=72, dtype=1, train=0):
        return lib.tops_gla_delta_bytes(
            struct.pack("=8q", nseq, chunks, nsegs, HV, K, V, dtype, train), back)

    # the state's 72 x 128 and the values' 72 x 64 elements of a chunk and head among them
    # where a backward follows
    assert size(0, train=1) - size(0) >= 6 * 2 * (72 * 128 + 72 * 64) and size(0) > 0
    assert size(1, train=1) >= 6 * 2 * (72 * 128 + 72 * 64)
    # and of three segments and two heads a state's 100 x 72 floats and a map's 128 x 128 pairs
    assert size(0, nsegs=3) - size(0) >= 6 * 4 * (100 * 72 + 128 * 128)
    assert size(1, nsegs=3) - size(1) >= 6 * 4 * 100 * 72
    assert not any(size(0, **bad) for bad in (
        dict(chunks=-1), dict(K=300), dict(V=0), dict(dtype=2), dict(nsegs=0), dict(HV=0)))
    assert lib.tops_gla_delta_bytes(None, 0) == 0


def test_segments():
    """Few columns in all are cut, many or short sequences are not."""
    f = _lib.load().tops_gla_delta_segment
    whole = 1 << 20
    assert f(1, 256, 16, 128) == 16 and f(2, 128, 16, 128) == 8
    assert f(1, 3, 1, 64) == whole and f(1, 12, 1, 64) == 2 and f(1, 256, 1, 64) == 8
    assert f(8, 1024, 32, 128) == whole and f(2, 128, 64, 128) == 32
    assert f(0, 0, 1, 64) == whole and f(1, 0, 1, 64) == whole
    assert f(1, 1 << 25, 1, 64) == 1 << 17


def test_segments_of_packed_sequences():
    """All segments at once where they fit, by the average where they do not, none of few chunks."""
    f = importlib.import_module("tops.ops.delta.gated_delta_rule")._segment
    for counts in ([28, 5, 33, 2, 47, 1, 8, 9], [30, 40, 50], [0, 256, 0], [7]):
        L = f(counts, 16)
        assert 2 <= L <= max(counts) / 2 and sum(-(-n // L) for n in counts) * 16 <= 256
    assert f([4] * 40 + [200], 16) == 23 and f([4] * 40, 16) == 4
    assert f([0, 0], 16) == 1 and f([3, 5, 1], 1) == 5 and f([60] * 16, 16) == 60


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("norm", [False, True])
def test_oracle_gradients_are_differences(norm):
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=F64)   # noqa: E731
    x = [r(1, 5, 1, 3), r(1, 5, 1, 3), r(1, 5, 2, 2), -r(1, 5, 2).abs(), r(1, 5, 2), r(2, 2, 3, 2)]
    x = [t.requires_grad_() for t in x]
    assert torch.autograd.gradcheck(lambda *a: delta(*a, cu=[0, 2, 5], l2norm=norm), x)


def test_oracle_norm_gradients_are_differences():
    gen = torch.Generator().manual_seed(0)
    x = [torch.randn(*s, generator=gen, dtype=F64).requires_grad_() for s in ((3, 5), (5,), (5,))]
    assert torch.autograd.gradcheck(ref_norm, x)
