"""qk_norm_rope against its formula in 64 bits.

Bounds: half a step of the output's type, and float32 roundings of a row's values: log2 D + 4 of
the mean square's sum and root, two products, and the rotation's (2 each for cos and sin, whose
angle is exact to half a step of a turn's fraction, 3.2 x 2^-24 of a radian). 24 roundings of the
row's largest normed value hold them all; a gradient goes through them twice, and a weight's adds
its terms in rows of at most tokens x heads."""

import pytest
import torch

from ssm_ref import close, qk
from tops.ops.rope import qk_norm_rope, rotary_inv_freq

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6


def make(B, T, Hq, Hk, D, dt, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)   # noqa: E731
    return dict(q=r(B, T, Hq, D).to(dt), k=(3 * r(B, T, Hk, D)).to(dt), q_weight=1 + 0.2 * r(D),
                k_weight=1 + 0.2 * r(D)), r


def check(x, freq, pos, inter, r, to=lambda n, t: t.to(DEV)):
    B, T, _, D = x["q"].shape
    d = {n: None if t is None else to(n, t).requires_grad_() for n, t in x.items()}
    out = qk_norm_rope(**d, inv_freq=None if freq is None else freq.to(DEV),
                       positions=None if pos is None else pos.to(DEV), eps=EPS, interleaved=inter)
    p = torch.arange(T).expand(B, T) if pos is None else pos.expand(B, T)
    ups = [r(*t.shape).to(x["q"].dtype) for t in out]
    names = [n for n, t in d.items() if t is not None]
    got = dict(zip(names, torch.autograd.grad(list(out), [d[n] for n in names],
                                              [u.to(DEV) for u in ups])))
    for n, o, up in zip(("q", "k"), out, ups):
        assert o.dtype == x[n].dtype and o.is_contiguous()
        ref = qk(x[n], x[n + "_weight"], freq, p, EPS, inter, up)
        close(n, o, ref["y"], ref["y"].abs().amax(-1, keepdim=True).expand(ref["y"].shape), 24)
        w = 1 if x[n + "_weight"] is None else x[n + "_weight"].abs().max().item()
        rstd = torch.rsqrt(x[n].double().square().mean(-1, keepdim=True) + EPS)
        m = x[n].double().abs() * rstd
        g = up.double().abs().amax(-1, keepdim=True) * 2   # a turned pair: at most sqrt(2) larger
        mag = (rstd * w * g * (1 + m * m.amax(-1, keepdim=True)))
        close("d" + n, got[n], ref["dx"], mag, 48)
        if n + "_weight" in got:
            close(f"d{n}_weight", got[n + "_weight"], ref["dw"], (g * m).sum((0, 1, 2)),
                  48 + B * T * x[n].shape[2])


@pytest.mark.parametrize("D", [2, 7, 16, 64, 70, 80, 96, 128, 200, 256, 512])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_head_sizes(D, inter, dt):
    x, r = make(2, 5, 3, 2, D, dt)
    check(x, rotary_inv_freq(D // 2 * 2), None, inter, r)


@pytest.mark.parametrize("D,R", [(128, 0), (128, 2), (128, 64), (96, 40), (70, 34), (64, 36), (9, 4)])
@pytest.mark.parametrize("inter", [False, True])
def test_partial_rotation(D, R, inter):
    x, r = make(1, 9, 2, 1, D, torch.bfloat16)
    check(x, rotary_inv_freq(R), None, inter, r)


@pytest.mark.parametrize("B,T,Hq,Hk", [(1, 1, 1, 1), (5, 1, 16, 4), (1, 3, 20, 5), (3, 7, 1, 9),
                                       (2, 2050, 3, 1)])
def test_heads_and_lengths(B, T, Hq, Hk):
    x, r = make(B, T, Hq, Hk, 32, torch.bfloat16)
    check(x, rotary_inv_freq(32), None, False, r)


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_positions(itype):
    x, r = make(2, 6, 2, 2, 64, torch.float32)
    pos = torch.tensor([[0, 1, 1 << 20, (1 << 31) - 1, 7, 3], [5, 5, 5, 131071, 99, 12345678]])
    check(x, rotary_inv_freq(64, 1e6), pos.to(itype), False, r)
    check(x, rotary_inv_freq(64), pos[1].to(itype), True, r)
    check(x, rotary_inv_freq(64), -pos.to(itype), False, r)


def test_far_positions_of_64_bits():
    x, r = make(1, 3, 1, 1, 64, torch.float32)
    # 2^33 at a frequency of 1: the 64-bit reference itself keeps 2^-20 of a radian
    check(x, rotary_inv_freq(64) * 2.0 ** -8, torch.tensor([1 << 33, (1 << 33) + 1, -(1 << 33)]),
          False, r)


@pytest.mark.parametrize("off", ["q_weight", "k_weight", "inv_freq"])
def test_optional_arguments(off):
    x, r = make(2, 5, 4, 2, 64, torch.bfloat16)
    if off != "inv_freq":
        x[off] = None
    check(x, None if off == "inv_freq" else rotary_inv_freq(64), None, False, r)


@pytest.mark.parametrize("pad", [0, 3])
def test_views_of_a_fused_projection(pad):
    x, r = make(2, 9, 4, 2, 64, torch.bfloat16)

    def view(n, t):
        t = t.to(DEV)
        if t.dim() < 4:
            return t.detach()
        wide = torch.full((2, 9, 8, 64 + pad), 5.0, dtype=t.dtype, device=DEV)
        v = wide[:, :, 1:1 + t.shape[2], pad:]
        v.copy_(t)
        return v.detach()

    check(x, rotary_inv_freq(64), None, False, r, view)
    check(x, rotary_inv_freq(64), None, False, r,   # heads before tokens, and no unit stride
          lambda n, t: (t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) if n == "q"
                        else t.to(DEV).transpose(-1, -2).contiguous().transpose(-1, -2)
                        if n == "k" else t.to(DEV)).detach())


def test_zero_rows_and_infinities():
    """A row of zeros stays zero (the norm's eps), with finite gradients; NaN and inf stay in
    their head."""
    x, r = make(1, 4, 3, 1, 64, torch.float32)
    x["q"][0, 1, 1] = 0
    check(x, rotary_inv_freq(64), None, False, r)
    x["q"][0, 2, 0, 5] = float("nan")
    x["q"][0, 3, 2, 9] = float("inf")
    d = {n: t.to(DEV) for n, t in x.items()}
    q, k = qk_norm_rope(**d, inv_freq=rotary_inv_freq(64, device=DEV))
    bad = ~torch.isfinite(q.cpu())
    assert bad[0, 2, 0].any() and bad[0, 3, 2].any() and torch.isfinite(k).all()
    bad[0, 2, 0] = bad[0, 3, 2] = False
    assert not bad.any()


def test_shared_weight():
    """One weight for queries and keys: its gradient is the sum of both."""
    x, r = make(1, 6, 2, 2, 32, torch.float32)
    d = {n: t.to(DEV) for n, t in x.items()}
    w = d["q_weight"].clone().requires_grad_()
    f = rotary_inv_freq(32, device=DEV)
    up = [r(1, 6, 2, 32), r(1, 6, 2, 32)]
    out = qk_norm_rope(d["q"], d["k"], w, w, f)
    got, = torch.autograd.grad(list(out), w, [u.to(DEV) for u in up])
    p = torch.arange(6)[None]
    refs = [qk(x[n], x["q_weight"], f, p, EPS, False, u) for n, u in zip("qk", up)]
    mag = sum(2 * u.double().abs().amax(-1, keepdim=True).expand(u.shape).sum((0, 1, 2)) * 6
              for u in up)
    close("dw", got, refs[0]["dw"] + refs[1]["dw"], mag, 48 + 24)


def test_directional_derivative():
    x, r = make(1, 5, 2, 1, 16, torch.float32)
    f = rotary_inv_freq(16)
    up = [r(1, 5, 2, 16), r(1, 5, 1, 16)]
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    out = qk_norm_rope(**d, inv_freq=f.to(DEV), eps=EPS)
    got = torch.autograd.grad(list(out), list(d.values()), [u.to(DEV) for u in up])
    p = torch.arange(5)[None]

    def value(s, n, v):
        z = {k: t.double() + (s * v if k == n else 0) for k, t in x.items()}
        return sum((qk(z[m], z[m + "_weight"], f, p, EPS, False)["y"] * u).sum().item()
                   for m, u in zip("qk", up))

    for n, g in zip(d, got):
        v = torch.randn(x[n].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(5))
        ref = (value(1e-5, n, v) - value(-1e-5, n, v)) / 2e-5
        t = g.cpu().double() * v
        assert abs(t.sum().item() - ref) <= 1e-5 * t.abs().sum().item(), n


def test_graph_and_unused_output():
    x, r = make(2, 9, 4, 2, 64, torch.bfloat16)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    f = rotary_inv_freq(64, device=DEV)
    up = r(2, 9, 4, 64).to(torch.bfloat16).to(DEV)

    def step():
        q, k = qk_norm_rope(**d, inv_freq=f)
        return [q.detach(), k.detach(), *torch.autograd.grad(q, [d["q"], d["k"], d["q_weight"]], up)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            d["q"].copy_(torch.randn(2, 9, 4, 64, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert (out[3] == 0).all()


def test_empty_calls():
    x, _ = make(2, 0, 4, 2, 64, torch.bfloat16)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    q, k = qk_norm_rope(**d, inv_freq=rotary_inv_freq(64, device=DEV))
    assert q.shape == (2, 0, 4, 64)
    g, = torch.autograd.grad(q, d["q_weight"], q.detach())
    assert (g == 0).all()


@pytest.mark.parametrize("D,R", [(130, 130), (256, 100), (200, 4), (258, 2), (512, 500), (384, 0),
                                 (257, 256), (512, 512)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_wide_heads(D, R, inter, dt):
    """More than 128 columns on aligned rows, with a rotated half that is no whole number of the
    lanes' pieces, and with one that is."""
    x, r = make(2, 5, 3, 2, D, dt)
    check(x, rotary_inv_freq(R), None, inter, r)
