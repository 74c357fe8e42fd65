"""Long and captured calls of the selective state space operators and of qk_norm_rope.

What a long call cuts into longer runs has the same arithmetic for every element as the short calls
that the other tests hold against 64-bit forms, so that its outputs are compared with theirs bit by
bit; sums over tokens are compared to float32 roundings, at most one a term."""

import pytest
import torch

import test_gpu_ssm_scan as scan_tests
from ssm_ref import close, conv
from tops.ops.rope import qk_norm_rope, rotary_inv_freq
from tops.ops.ssm import causal_conv1d, selective_scan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("lens", [None, [8000, 1, 0, 999]])
def test_scan_of_hundreds_of_pieces(lens):
    """More pieces than a thread of the fold takes in one run; slow decay carries the states."""
    cu = None
    if lens:
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
    x, r = scan_tests.make(1, 9000, 6, 5, torch.float32, S=len(lens) if lens else 1)
    x["A"] = x["A"] * 1e-2
    scan_tests.check(x, True, cu, True, r)


def test_scan_state_that_is_forgotten_at_once():
    """A of -inf: exp(delta A) is 0, also for the tokens past a piece's end."""
    x, _ = scan_tests.make(2, 77, 20, 16, torch.float32)
    x["A"][:, 3] = float("-inf")
    scan_tests.check(x, True, None, False, None)


def test_scan_infinite_last_token():
    """An infinity at a sequence's last token is in its state as such: nothing after it makes a
    NaN of it, and the other states and the next sequence do not see it."""
    x, _ = scan_tests.make(1, 74, 20, 16, torch.float32, S=2)
    cu = [0, 37, 74]
    x["B"][0, 36, 2] = float("inf")
    x["C"][0, 36, 2] = 1.0
    d = {n: t.to(DEV) for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True, cu_seqlens=cu)
    y, ht = y.cpu(), ht.cpu()
    ref, mag = scan_tests.reference(x, True, cu)
    assert torch.equal(ht[0, :, 2].double(), ref["ht"][0, :, 2]) and torch.isinf(ht[0, :, 2]).all()
    keep = [n for n in range(16) if n != 2]
    close("ht", ht[0][:, keep], ref["ht"][0][:, keep], mag["ht"][0][:, keep], 4 * 37 + 64)
    close("ht", ht[1], ref["ht"][1], mag["ht"][1], 4 * 37 + 64)
    rest = [t for t in range(74) if t != 36]
    close("y", y[:, rest], ref["y"][:, rest], mag["y"][:, rest], 4 * 74 + 64)
    assert torch.equal(y[0, 36].double(), ref["y"][0, 36])


def test_conv_long_runs():
    B, T, D, W = 1, 40000, 4096, 4
    gen = torch.Generator(device=DEV).manual_seed(0)
    x, dy = (torch.randn(B, T, D, generator=gen, device=DEV).bfloat16() for _ in range(2))
    w = (0.5 * torch.randn(D, W, generator=gen, device=DEV)).bfloat16().requires_grad_()
    x.requires_grad_()
    y, ht = causal_conv1d(x, w, None, "silu", output_final_state=True)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    state, terms = None, torch.zeros(D, W, dtype=torch.float64, device=DEV)
    edges = [0, 5, 300, 9000, 9001, 25000, T]
    for a, b in zip(edges, edges[1:]):
        yy, state = causal_conv1d(x[:, a:b], w, None, "silu", initial_state=state,
                                  output_final_state=True)
        assert torch.equal(yy, y[:, a:b])
        # gradients of a piece's inputs from its own tokens: all but those of its last rows
        gx, gw = torch.autograd.grad(yy, [x, w], dy[:, a:b], retain_graph=True)
        assert torch.equal(gx[:, a:max(a, b - W + 1)], dx[:, a:max(a, b - W + 1)])
        terms += gw.double()
    assert torch.equal(state, ht)
    # six sums, each rounded to bfloat16, and the whole one
    assert ((terms - dw.double()).abs() <= 7 * 2.0 ** -8 * terms.abs().clamp(min=dw.abs().max().item())).all()


@pytest.mark.parametrize("xt,wt", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("D", [24, 13])
def test_conv_mixed_types(xt, wt, D):
    gen = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(2, 40, D, generator=gen).to(xt) for _ in range(2))
    w, b = (0.5 * torch.randn(D, 4, generator=gen)).to(wt), torch.randn(D, generator=gen).to(wt)
    d = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y, _ = causal_conv1d(*d, activation="silu")
    ref, mag = [conv(x, w, b, True, None, None, dy, mag=m) for m in (False, True)]
    close("y", y, ref["y"], mag["y"], 13)
    for n, g, t in zip(("x", "weight", "bias"), torch.autograd.grad(y, d, dy.to(DEV)), d):
        assert g.dtype == t.dtype
        close(n, g, ref["d" + n], mag["d" + n], 30 + 80)


def test_qk_many_tokens():
    T, Hq, Hk, D = 33001, 5, 3, 16
    gen = torch.Generator(device=DEV).manual_seed(0)
    qkv = torch.randn(1, T, Hq + 2 * Hk, D, generator=gen, device=DEV).bfloat16()
    q, k = qkv[:, :, :Hq].requires_grad_(), qkv[:, :, Hq:Hq + Hk].requires_grad_()
    w = [(1 + 0.1 * torch.randn(D, generator=gen, device=DEV)).requires_grad_() for _ in range(2)]
    ups = [torch.randn(1, T, h, D, generator=gen, device=DEV).bfloat16() for h in (Hq, Hk)]
    freq = rotary_inv_freq(8, device=DEV)
    pos = torch.arange(T, device=DEV) * 7
    out = qk_norm_rope(q, k, *w, freq, pos)
    got = torch.autograd.grad(out, [q, k, *w], ups)
    sums = [torch.zeros(D, dtype=torch.float64, device=DEV) for _ in range(2)]
    size = [torch.zeros(D, dtype=torch.float64, device=DEV) for _ in range(2)]
    for a, b in ((0, 1), (1, 700), (700, 16000), (16000, 16003), (16003, T)):
        o = qk_norm_rope(q[:, a:b], k[:, a:b], *w, freq, pos[a:b])
        g = torch.autograd.grad(o, [q, k, *w], [u[:, a:b] for u in ups])
        for i in range(2):
            assert torch.equal(o[i], out[i][:, a:b]) and torch.equal(g[i][:, a:b], got[i][:, a:b])
            sums[i] += g[2 + i].double()
    for i, t in enumerate((q, k)):
        m = t.detach().double()
        m = m.abs() * torch.rsqrt(m.square().mean(-1, keepdim=True) + 1e-6)
        size[i] = (m * ups[i].double().abs().amax(-1, keepdim=True) * 2).sum((0, 1, 2))
        err = (got[2 + i].double() - sums[i]).abs()
        assert (err <= 2 * T * t.shape[2] * 2.0 ** -24 * size[i]).all()


def test_packed_sequences_in_a_graph():
    """The tables of a captured call stay, whatever other lengths come after it; lengths that were
    never run cannot be captured and say so."""
    gen = torch.Generator(device=DEV).manual_seed(0)
    D, N, cu = 64, 16, [0, 100, 101, 300]
    x = {n: torch.randn(*s, generator=gen, device=DEV) for n, s in
         (("u", (1, 300, D)), ("delta", (1, 300, D)), ("B", (1, 300, N)), ("C", (1, 300, N)))}
    A = -torch.rand(D, N, generator=gen, device=DEV)
    w = torch.randn(D, 4, generator=gen, device=DEV)

    def step(offsets):
        u, window = causal_conv1d(x["u"], w, None, "silu", output_final_state=True,
                                  cu_seqlens=offsets)
        y, h = selective_scan(u, x["delta"], A, x["B"], x["C"], delta_softplus=True,
                              output_final_state=True, cu_seqlens=offsets)
        return y, h, window

    with torch.no_grad():
        step(cu)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cu)
        for k in range(70):   # more lengths than are kept
            step([0, 5 + k, 300])
        junk = [torch.full((256,), 1 << 30, dtype=torch.int32, device=DEV) for _ in range(200)]
        for k in range(3):
            for t in x.values():
                t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            want = step(cu)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        del junk
        other = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="capture"):
            with torch.cuda.graph(other):
                step([0, 7, 300])


def test_scan_of_uncut_sequences():
    """A batch that fills the device is not cut into pieces: the same values as a few of its rows,
    which are cut, to float32 roundings (an output's sum has the state of up to 200 tokens before
    it, each good to 4 roundings of the largest magnitude)."""
    B, T, D, N = 256, 200, 512, 16
    x, r = scan_tests.make(B, T, D, N, torch.float32)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True)
    dy = r(B, T, D).to(DEV)
    names = ["u", "delta", "z", "B", "C", "initial_state"]
    got = torch.autograd.grad(y, [d[n] for n in names], dy)
    rows = [0, 101, 255]
    ref, mag = scan_tests.reference({n: t[rows] if t.shape[0] == B else t for n, t in x.items()},
                                    True, None, dy[rows].cpu(), torch.zeros(3, D, N))
    terms = 4 * T + 64
    close("y", y[rows], ref["y"], mag["y"], terms)
    close("ht", ht[rows], ref["ht"], mag["ht"], terms)
    for n, g in zip(names, got):
        close("d" + n, g[rows], ref["d" + n], mag["d" + n], terms + T + D)


def test_scan_of_many_packed_sequences():
    """More sequences than one dimension of the fold's grid could hold with 64 states of 1024
    channels, one of them cut into pieces: the short ones have their own values, bit by bit."""
    S, D, N, first = 16400, 1024, 64, 600
    T = first + S
    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)   # noqa: E731
    x = dict(u=r(1, T, D), delta=r(1, T, D), B=r(1, T, N), C=r(1, T, N))
    A, dy = -torch.rand(D, N, generator=gen, device=DEV), r(1, T, D)
    cu = [0, *range(first, T + 1)]

    def run(x, dy, cu):
        x = {n: t.detach().requires_grad_() for n, t in x.items()}
        y, _ = selective_scan(x["u"], x["delta"], A, x["B"], x["C"], delta_softplus=True,
                              cu_seqlens=cu)
        return [y.detach(), *torch.autograd.grad(y, list(x.values()), dy)]

    alone = {n: t[0, first:].unsqueeze(1) for n, t in x.items()}
    want = run(alone, dy[0, first:].unsqueeze(1), None)
    for a, b in zip(run(x, dy, cu), want):
        assert torch.equal(a[0, first:], b.squeeze(1))


def far(t, buf, at):
    """t's rows 2^26 elements apart in `buf`, from column `at` on: the last ones past 2^31."""
    v = buf[at:].as_strided(t.shape, (0, (1 << 26) + 8, *t.stride()[2:]))
    v.copy_(t)
    return v


def test_offsets_past_32_bits():
    T, D, N = 40, 136, 16
    gen = torch.Generator(device=DEV).manual_seed(0)
    buf = torch.empty(T * ((1 << 26) + 8) + 4096, dtype=torch.bfloat16, device=DEV)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV).bfloat16()   # noqa: E731
    near = {n: r(1, T, D) for n in ("u", "delta", "z", "dy")} | {n: r(1, T, N) for n in ("B", "C")}
    A, w = -torch.rand(D, N, generator=gen, device=DEV), r(D, 4)
    freq = rotary_inv_freq(8, device=DEV)
    x = {n: far(t, buf, 256 * i) for i, (n, t) in enumerate(near.items())}
    got, want = [], []
    for out, v in ((want, near), (got, x)):
        v = {n: t.detach().requires_grad_(n != "dy") for n, t in v.items()}
        y, _ = selective_scan(v["u"], v["delta"], A, v["B"], v["C"], z=v["z"], delta_softplus=True)
        out += [y, *torch.autograd.grad(y, [v[n] for n in ("u", "delta", "z", "B", "C")], v["dy"])]
        y, _ = causal_conv1d(v["u"], w, None, "silu")
        out += [y, *torch.autograd.grad(y, [v["u"]], v["dy"])]
        q, k, dq = (v[n].unflatten(2, (17, 8)) for n in ("u", "delta", "dy"))
        o = qk_norm_rope(q, k, None, None, freq)
        out += [*o, *torch.autograd.grad(o, [q, k], [dq, dq])]
    assert x["C"].data_ptr() + 2 * x["C"].stride(1) * (T - 1) - buf.data_ptr() > 1 << 32
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_slots_past_32_bits():
    from tops.ops.ssm import causal_conv1d_step, selective_scan_step

    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)   # noqa: E731
    D, N, W = 2048, 16, 4
    slots = torch.tensor([70000, 3, 65536], dtype=torch.int64, device=DEV)   # times 2^15 floats
    few = torch.arange(3, device=DEV)
    small, pool = r(3, D, N), torch.empty(70001, D, N, device=DEV)
    pool[slots] = small
    a = [r(3, D), r(3, D), -torch.rand(D, N, generator=gen, device=DEV), r(3, N), r(3, N)]
    assert torch.equal(selective_scan_step(pool, *a, delta_softplus=True, state_indices=slots),
                       selective_scan_step(small, *a, delta_softplus=True, state_indices=few))
    assert torch.equal(pool[slots], small)
    del pool
    slots = slots * 8   # times 2^13 elements
    small, pool = r(3, W, D).bfloat16(), torch.empty(560001, W, D, dtype=torch.bfloat16, device=DEV)
    pool[slots] = small
    x, w = r(3, D).bfloat16(), r(D, W)
    assert torch.equal(causal_conv1d_step(x, pool, w, state_indices=slots),
                       causal_conv1d_step(x, small, w, state_indices=few))
    assert torch.equal(pool[slots], small)
