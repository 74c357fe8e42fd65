"""causal_conv1d and causal_conv1d_step against the convolution in 64 bits.

Bounds: half a step of the output's type, and the float32 roundings of the sums: W + 1 products
and additions of z and about 8 of the activation (exponential, reciprocal, products); twice that
for a gradient, which goes through both; the weights' sums add one a token at most."""

import pytest
import torch

from ssm_ref import close, conv
from tops.modules import ShortConvolution
from tops.ops.ssm import causal_conv1d, causal_conv1d_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(B, T, D, W, dt, S=None, bias=True, init=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)   # noqa: E731
    return dict(x=r(B, T, D).to(dt), weight=(0.5 * r(D, W)).to(dt),
                bias=(0.3 * r(D)).to(dt) if bias else None,
                initial_state=r(B if S is None else S, W, D).to(dt) if init else None), r


def check(x, act, cu, r, to=lambda n, t: t.to(DEV), shape=None):
    dt = x["x"].dtype
    B, T, D = x["x"].shape
    W = x["weight"].shape[-1]
    d = {n: None if t is None else to(n, t).requires_grad_() for n, t in x.items()}
    if shape:
        d["weight"] = d["weight"].detach().reshape(shape).requires_grad_()
    y, ht = causal_conv1d(**d, activation=act, output_final_state=True, cu_seqlens=cu)
    assert y.dtype == dt and ht.dtype == dt
    dy, dht = r(B, T, D).to(dt), r(*ht.shape).to(dt)
    ref, mag = [conv(x["x"], x["weight"], x["bias"], act is not None, x["initial_state"], cu, dy,
                     dht, mag=m) for m in (False, True)]
    close("y", y, ref["y"], mag["y"], W + 9)
    assert torch.equal(ht.cpu().double(), ref["ht"])
    names = [n for n, t in d.items() if t is not None]
    got = torch.autograd.grad([y, ht], [d[n] for n in names], [dy.to(DEV), dht.to(DEV)])
    for n, t in zip(names, got):
        assert t.dtype == d[n].dtype and t.shape == d[n].shape
        many = B * T if n in ("weight", "bias") else 0
        close("d" + n, t.reshape(ref["d" + n].shape), ref["d" + n], mag["d" + n],
              2 * (W + 9) + W + many)


# tokens around a run (8, 16) and its rows in flight, channels around a vector and a slab (512)
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 3, 8), (1, 8, 520), (2, 33, 24), (3, 70, 17),
                                   (1, 129, 64), (2, 1100, 36)])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_forward_backward(B, T, D, act, dt):
    x, r = make(B, T, D, 4, dt)
    check(x, act, None, r)


@pytest.mark.parametrize("W", [1, 2, 3, 5, 6, 7, 8])
@pytest.mark.parametrize("D", [40, 13])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_widths(W, D, dt):
    x, r = make(2, 19, D, W, dt)
    check(x, "silu", None, r)


@pytest.mark.parametrize("off", ["bias", "init"])
def test_optional_arguments(off):
    x, r = make(2, 40, 16, 4, torch.bfloat16, **{off: False})
    check(x, "swish", None, r)


@pytest.mark.parametrize("lens", [[1], [2, 1, 3, 30], [0, 7, 0, 0, 65, 0], [0, 0], [3, 3, 3, 100]])
@pytest.mark.parametrize("init", [True, False])
def test_packed(lens, init):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x, r = make(1, cu[-1], 24, 4, torch.float32, S=len(lens), init=init)
    check(x, "silu", cu, r)


def test_long_runs():
    """Enough tokens for the longest runs, with boundaries inside them."""
    cu = [0, 5000, 5001, 12345, 16500]
    x, r = make(1, 16500, 8, 4, torch.float32, S=4)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = causal_conv1d(**d, activation="silu", output_final_state=True, cu_seqlens=cu)
    dy = r(1, 16500, 8)
    got = dict(zip(d, torch.autograd.grad(y, list(d.values()), dy.to(DEV))))
    for s, (a, b) in enumerate(zip(cu, cu[1:])):   # the ends of each sequence
        for lo, hi in ((a, min(b, a + 70)), (max(a, b - 70), b)):
            w0 = max(a, lo - 3)
            first = x["initial_state"][s:s + 1] if lo == a else torch.cat(
                [torch.zeros(1, 4 - (lo - w0), 8), x["x"][:, w0:lo]], 1)
            cut = x["x"][:, lo:min(b, hi + 3)], x["weight"], x["bias"], True, first
            ref, mag = [conv(*cut, dy=dy[:, lo:min(b, hi + 3)], mag=m) for m in (False, True)]
            n = hi - lo
            close("y", y[:, lo:hi], ref["y"][:, :n], mag["y"][:, :n], 13)
            close("dx", got["x"][:, lo:hi], ref["dx"][:, :n], mag["dx"][:, :n], 30)
    with torch.no_grad():   # the weights' gradient over all tokens, in 64 bits
        p = torch.cat([torch.cat([x["initial_state"][s, 1:], x["x"][0, a:b]])
                       .unfold(0, 4, 1) for s, (a, b) in enumerate(zip(cu, cu[1:]))]).double()
        z = (p * x["weight"].double()).sum(-1) + x["bias"].double()
        sg = torch.sigmoid(z)
        dz = dy[0].double() * sg * (1 + z * (1 - sg))
        dw, m = (dz[..., None] * p).sum(0), (2 * dy[0].double().abs()[..., None] * (1 + p.abs())).sum(0)
    # partial sums of 64 tokens in a row, then of the runs: far fewer roundings in a row than
    # tokens, 64 + the runs' count / 4 + those of a term
    close("dweight", got["weight"], dw, m, 64 + 65 + 30)


def test_strided_views():
    x, r = make(2, 40, 24, 4, torch.bfloat16)

    def view(n, t):
        t = t.to(DEV)
        if n == "x":
            return torch.cat([t, t], -1)[..., 24:].detach()
        return t.detach()

    check(x, "silu", None, r, view)
    check(x, "silu", None, r, lambda n, t: (torch.cat([t[..., :1], t], -1).to(DEV)[..., 1:]
                                            if n == "x" else t.to(DEV)).detach())
    check(x, "silu", None, r, shape=(24, 1, 4))


def test_final_state_is_the_layers_cache():
    """ShortConvolution's cache and this operator's state are the same thing."""
    m = ShortConvolution(32, 4, bias=True, rngs=3, device=DEV)
    x, _ = make(2, 21, 32, 4, torch.float32, init=False)
    xx = x["x"].to(DEV)
    with torch.no_grad():
        y0, c0 = m(xx, output_final_state=True)
        y1, c1 = causal_conv1d(xx, m.weight, m.bias, "silu", output_final_state=True)
    assert torch.equal(c0, c1)
    ref, mag = [conv(xx, m.weight, m.bias, True, mag=k) for k in (False, True)]
    close("y", y1, ref["y"], mag["y"], 13)


def test_pieces_equal_the_whole():
    """Run piece by piece with the state carried on: the same bits."""
    x, _ = make(2, 90, 48, 4, torch.bfloat16)
    d = {n: t.to(DEV) for n, t in x.items()}
    y, ht = causal_conv1d(**d, activation="silu", output_final_state=True)
    h, ys = d["initial_state"], []
    for a, b in ((0, 1), (1, 3), (3, 40), (40, 90)):
        yy, h = causal_conv1d(d["x"][:, a:b], d["weight"], d["bias"], "silu", h, True)
        ys.append(yy)
    assert torch.equal(torch.cat(ys, 1), y) and torch.equal(h, ht)


def test_directional_derivative():
    x, r = make(2, 21, 6, 4, torch.float32)
    dy, dht = r(2, 21, 6), r(2, 4, 6)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = causal_conv1d(**d, activation="silu", output_final_state=True)
    got = torch.autograd.grad([y, ht], list(d.values()), [dy.to(DEV), dht.to(DEV)])

    def value(s, n, v):
        z = {k: t.double() + (s * v if k == n else 0) for k, t in x.items()}
        o = conv(z["x"], z["weight"], z["bias"], True, z["initial_state"])
        return ((o["y"] * dy).sum() + (o["ht"] * dht).sum()).item()

    for n, g in zip(d, got):
        v = torch.randn(x[n].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(5))
        ref = (value(1e-4, n, v) - value(-1e-4, n, v)) / 2e-4
        p = g.cpu().double() * v
        assert abs(p.sum().item() - ref) <= 1e-5 * p.abs().sum().item(), n


def test_nan_stays_in_its_window():
    x, _ = make(1, 40, 16, 4, torch.bfloat16)
    x["x"][0, 10, 3] = float("nan")
    d = {n: t.to(DEV) for n, t in x.items()}
    y, _ = causal_conv1d(**d, activation="silu")
    bad = torch.isnan(y.cpu())
    want = torch.zeros_like(bad)
    want[0, 10:14, 3] = True
    assert torch.equal(bad, want)


def test_graph():
    x, r = make(2, 50, 32, 4, torch.bfloat16)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    dy = r(2, 50, 32).to(torch.bfloat16).to(DEV)

    def step():
        y, ht = causal_conv1d(**d, activation="silu", output_final_state=True)
        return [y.detach(), ht.detach(), *torch.autograd.grad(y, list(d.values()), dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            d["x"].copy_(torch.randn(2, 50, 32, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_empty_calls():
    x, _ = make(2, 0, 24, 4, torch.float32)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = causal_conv1d(**d, activation="silu", output_final_state=True)
    assert y.shape == (2, 0, 24) and torch.equal(ht, d["initial_state"])
    g = torch.autograd.grad(ht, [d["initial_state"], d["weight"]], torch.ones_like(ht))
    assert (g[0] == 1).all() and (g[1] == 0).all()


# ---------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,D,W", [(1, 1, 1), (3, 20, 4), (5, 257, 4), (2, 48, 8), (130, 1024, 3)])
@pytest.mark.parametrize("act", [None, "silu"])
def test_step(B, D, W, dt, act):
    x, _ = make(B, 1, D, W, dt)
    ref, mag = [conv(x["x"], x["weight"], x["bias"], act is not None, x["initial_state"], mag=m)
                for m in (False, True)]
    state = x["initial_state"].to(DEV)
    wide = torch.cat([x["x"][:, 0], x["x"][:, 0]], -1).to(DEV)
    y = causal_conv1d_step(wide[:, :D], state, x["weight"].to(DEV), x["bias"].to(DEV), act)
    close("y", y[:, None], ref["y"], mag["y"], W + 9)
    assert torch.equal(state.cpu().double(), ref["ht"])


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_step_slots(itype):
    B, D, W = 5, 24, 4
    x, r = make(B, 1, D, W, torch.bfloat16)
    pool = r(7, W, D).to(torch.bfloat16)
    slots = torch.tensor([6, -1, 0, 7, 3], dtype=itype)
    ref, mag = [conv(x["x"], x["weight"], x["bias"], True, pool[slots.clamp(0, 6).long()], mag=m)
                for m in (False, True)]
    dev = pool.to(DEV)
    y = causal_conv1d_step(x["x"][:, 0].to(DEV), dev, x["weight"].to(DEV).float(), x["bias"].to(DEV),
                           "silu", slots.to(DEV))
    live = [0, 2, 4]
    close("y", y[live], ref["y"][live, 0], mag["y"][live, 0], W + 9)
    assert (y[[1, 3]] == 0).all()
    assert torch.equal(dev[[6, 0, 3]].cpu().double(), ref["ht"][live])
    rest = [1, 2, 4, 5]
    assert torch.equal(dev[rest].cpu(), pool[rest])


def test_steps_equal_the_convolution():
    x, _ = make(2, 30, 40, 4, torch.bfloat16)
    d = {n: t.to(DEV) for n, t in x.items()}
    y, ht = causal_conv1d(**d, activation="silu", output_final_state=True)
    state = d["initial_state"].clone()
    ys = [causal_conv1d_step(d["x"][:, t], state, d["weight"], d["bias"], "silu") for t in range(30)]
    assert torch.equal(torch.stack(ys, 1), y) and torch.equal(state, ht)


def test_step_of_a_state_that_a_backward_needs():
    """The step counts as an in-place operation on its state: a convolution that kept it for its
    backward says so instead of using the new values. States without a counter work as before."""
    x, r = make(2, 9, 24, 4, torch.float32)
    d = {n: t.to(DEV) for n, t in x.items()}
    pool = d["initial_state"]
    w = d["weight"].requires_grad_()
    y, _ = causal_conv1d(d["x"], w, d["bias"], "silu", initial_state=pool)
    version = pool._version
    with torch.no_grad():
        causal_conv1d_step(d["x"][:, 0], pool, w, d["bias"], "silu")
    assert pool._version > version
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    with torch.inference_mode():
        state = pool.clone()
        assert state.is_inference()
        want = causal_conv1d_step(d["x"][:, 1], pool, w, d["bias"], "silu")
        assert torch.equal(causal_conv1d_step(d["x"][:, 1], state, w, d["bias"], "silu"), want)
        assert torch.equal(state, pool)


@pytest.mark.parametrize("D", [4096, 4099])
def test_packed_sequences_in_long_runs(D):
    """Runs of 128 tokens with the boundaries of sequences inside them, at their first and last
    token and in the rows that a run reads past its end; the weights' and the bias's gradients to
    float32 roundings, for a part of the channels."""
    T, W = 40000, 4
    cu = [0, 1, 128, 130, 131, 131, 253, 256, 257, 511, 515, 20000, 20479, 20480, 20607, 32768, T]
    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)   # noqa: E731
    x, dy = r(1, T, D).bfloat16(), r(1, T, D).bfloat16()
    w, b, init = 0.5 * r(D, W), 0.3 * r(D), r(len(cu) - 1, W, D).bfloat16()
    leaves = [t.requires_grad_() for t in (x, w, b, init)]
    y, ht = causal_conv1d(x, w, b, "silu", init, True, cu)
    dx, dw, db, di = torch.autograd.grad(y, leaves, dy)
    cols = torch.cat([torch.arange(6), torch.arange(D // 2, D // 2 + 6), torch.arange(D - 9, D)])
    cols = cols.to(DEV)
    cut = lambda t, dim: t.detach().index_select(dim, cols).double()   # noqa: E731
    X, G, K, S = cut(x, 2)[0], cut(dy, 2)[0], cut(w, 0), cut(init, 2)
    rows = torch.cat([torch.cat([S[s], X[a:e]]) for s, (a, e) in enumerate(zip(cu, cu[1:]))])
    first = torch.repeat_interleave(torch.arange(1, len(cu), device=DEV) * W,
                                    torch.tensor(cu, device=DEV).diff())
    at = first + torch.arange(T, device=DEV)   # a token's row in `rows`, W more a sequence
    p = torch.stack([rows[at - W + 1 + j] for j in range(W)], -1)   # [T, cols, W]
    z = (p * K).sum(-1) + cut(b, 0)
    zm = (p.abs() * K.abs()).sum(-1) + cut(b, 0).abs()
    sg = torch.sigmoid(z)
    close("y", cut(y, 2)[0].to(y.dtype), (z * sg).cpu(), (1.1 * zm).cpu(), W + 9)
    dz, dzm = G * sg * (1 + z * (1 - sg)), G.abs() * (1.1 + 0.5 * zm)
    # sums of 128 tokens in a row, of four runs, then of a column's T / 512 partial sums by eight
    # threads, and the roundings of a term
    many = 128 + 4 + T // 512 // 8 + 1 + 8 + 2 * (W + 9)
    close("dweight", dw.index_select(0, cols), (dz[..., None] * p).sum(0).cpu(),
          (dzm[..., None] * p.abs()).sum(0).cpu(), many)
    close("dbias", db.index_select(0, cols), dz.sum(0).cpu(), dzm.sum(0).cpu(), many)
    back, mag = torch.zeros_like(rows), torch.zeros_like(rows)
    for j in range(W):
        back.index_add_(0, at - W + 1 + j, dz * K[:, j])
        mag.index_add_(0, at - W + 1 + j, dzm * K[:, j].abs())
    close("dx", dx.index_select(2, cols)[0], back[at].cpu(), mag[at].cpu(), 2 * (W + 9) + W)
    first = torch.tensor([c + W * s for s, c in enumerate(cu[:-1])], device=DEV)
    at = first[:, None] + torch.arange(W, device=DEV)
    close("dinit", di.index_select(2, cols), back[at].cpu(), mag[at].cpu(), 2 * (W + 9) + W)
    end = torch.tensor([c + W * s for s, c in enumerate(cu[1:])], device=DEV)
    assert torch.equal(cut(ht, 2), rows[end[:, None] + torch.arange(W, device=DEV)])
