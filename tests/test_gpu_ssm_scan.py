"""selective_scan and selective_scan_step against the recurrence in 64 bits.

Bounds: an output is off by at most half a step of its type, and by the float32 roundings of what
went into it. A state's factor exp(delta A) carries about 4 roundings (delta's softplus, A's and
the product's scaling to base 2, the exponential) each time, and its memory is at most the
sequence, so the terms' sums are good to 4 T + 64 roundings (64: the sums over states, pieces and
the output's own products); sums over channels or tokens add their count's order, log2 of it for
pairwise parts, at most the terms of one lane in a row (T)."""

import pytest
import torch

from ssm_ref import close, scan
from tops.ops.ssm import selective_scan, selective_scan_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(B, T, D, N, dt, seed=0, G=None, S=None, z=True, skip=True, bias=True, h0=True,
         softplus=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)   # noqa: E731
    g = (B, T, N) if G is None else (B, T, G, N)
    x = dict(u=r(B, T, D).to(dt), delta=(0.7 * r(B, T, D) if softplus
                                         else 0.1 * r(B, T, D).abs()).to(dt),
             A=-torch.exp(0.5 * r(D, N)) * torch.arange(1, N + 1) / 4, B=r(*g).to(dt),
             C=r(*g).to(dt))
    x["D"] = r(D) if skip else None
    x["z"] = r(B, T, D).to(dt) if z else None
    # without softplus a step size stays positive: a negative one grows the state without bound
    x["delta_bias"] = None if not bias else r(D) - 2.0 if softplus else 0.1 * r(D).abs()
    x["initial_state"] = r(B if S is None else S, D, N) if h0 else None
    return x, r


def reference(x, softplus, cu, dy=None, dht=None):
    y = dict(x)
    h0 = y.pop("initial_state")
    return [scan(**y, softplus=softplus, h0=h0, cu=cu, dy=dy, dht=dht, mag=m)
            for m in (False, True)]


def check(x, softplus, cu, grads, r, to=lambda n, t: t.to(DEV)):
    dt = x["u"].dtype
    B, T, D = x["u"].shape
    dx = {n: None if t is None else to(n, t).requires_grad_(grads) for n, t in x.items()}
    y, ht = selective_scan(**dx, delta_softplus=softplus, output_final_state=True, cu_seqlens=cu)
    assert y.dtype == dt and ht.dtype == torch.float32
    dy = dht = None
    if grads:
        dy, dht = r(B, T, D).to(dt), r(*ht.shape)
    ref, mag = reference(x, softplus, cu, dy, dht)
    terms = 4 * T + 64
    close("y", y, ref["y"], mag["y"], terms)
    close("ht", ht, ref["ht"], mag["ht"], terms)
    if not grads:
        return
    names = [n for n, t in dx.items() if t is not None]
    got = torch.autograd.grad([y, ht], [dx[n] for n in names], [dy.to(DEV), dht.to(DEV)])
    for n, t in zip(names, got):
        assert t.dtype == x[n].dtype and t.shape == x[n].shape
        close("d" + n, t, ref["d" + n], mag["d" + n], terms + B * T + D)


# tokens around a tile and a piece (16 and 64), channels around a block (128), odd ones
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 15, 8), (1, 16, 128), (3, 17, 130), (2, 64, 20),
                                   (1, 65, 256), (2, 200, 37), (1, 333, 136)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_forward_backward(B, T, D, dt):
    x, r = make(B, T, D, 16, dt)
    check(x, True, None, True, r)


@pytest.mark.parametrize("N", [1, 3, 8, 13, 17, 32, 33, 64])
def test_state_sizes(N):
    x, r = make(2, 70, 72, N, torch.bfloat16)
    check(x, True, None, True, r)


@pytest.mark.parametrize("G,D,N", [(1, 24, 16), (2, 260, 16), (4, 24, 20), (3, 9, 40)])
def test_groups(G, D, N):
    x, r = make(2, 67, D, N, torch.float32, G=G)
    check(x, True, None, True, r)


@pytest.mark.parametrize("off", ["z", "skip", "bias", "h0", "softplus"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_optional_arguments(off, dt):
    x, r = make(2, 81, 48, 16, dt, **{off: False})
    check(x, off != "softplus", None, True, r)


@pytest.mark.parametrize("lens", [[1], [5, 1, 64, 130], [0, 7, 0, 0, 65, 0], [0, 0], [16, 48, 300]])
def test_packed(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x, r = make(1, cu[-1], 40, 16, torch.float32, S=len(lens))
    check(x, True, cu, True, r)


def test_strided_views():
    """u, z, B and C as columns of wider projections, transposed ones copied."""
    x, r = make(2, 70, 40, 16, torch.bfloat16)

    def view(n, t):
        t = t.to(DEV)
        if n in ("u", "z", "B", "C"):
            pad = torch.full((*t.shape[:-1], 3), 7.0, dtype=t.dtype, device=DEV)
            return torch.cat([pad, t, pad], -1)[..., 3:-3].detach()
        if n == "delta":
            return t.transpose(1, 2).contiguous().transpose(1, 2).detach()
        return t.detach()

    check(x, True, None, True, r, view)


def test_broadcast_inputs():
    """One B and C for the whole batch, one u for all tokens: the gradients of the expanded views."""
    x, r = make(3, 40, 24, 8, torch.float32)
    for n in ("B", "C"):
        x[n] = x[n][:1].expand(3, -1, -1)
    x["u"] = x["u"][:, :1].expand(-1, 40, -1)
    check(x, True, None, True, r, lambda n, t: t.to(DEV).detach() if n not in ("u", "B", "C") else
          (t[:, :1].to(DEV).expand(-1, 40, -1) if n == "u" else t[:1].to(DEV).expand(3, -1, -1)))


def test_many_pieces_carry_the_state():
    """A long sequence of slow decay: every piece's entry state comes through all before it."""
    x, r = make(1, 1500, 8, 16, torch.float32)
    x["A"] = x["A"] * 1e-3
    check(x, True, None, True, r)


def test_pieces_equal_the_whole():
    """A prompt run piece by piece gives the same values, to float32 roundings."""
    x, _ = make(2, 230, 64, 16, torch.float32)
    d = {n: t.to(DEV) for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True)
    h, ys = d["initial_state"], []
    for a, b in ((0, 1), (1, 100), (100, 230)):
        cut = {n: t[:, a:b] if t.dim() == 3 and n != "initial_state" else t for n, t in d.items()}
        cut["initial_state"] = h
        yy, h = selective_scan(**cut, delta_softplus=True, output_final_state=True)
        ys.append(yy)
    ref, mag = reference(x, True, None)
    for name, t in (("y", torch.cat(ys, 1)), ("ht", h)):
        close(name, t, ref[name], mag[name], 4 * 230 + 64)


def test_directional_derivative():
    """<gradient, v> against central differences of the 64-bit recurrence (error of the
    differences: 1e-4^2 of the third derivative, far below the bound)."""
    x, r = make(1, 33, 12, 8, torch.float32)
    dy, dht = r(1, 33, 12), r(1, 12, 8)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True)
    got = torch.autograd.grad([y, ht], list(d.values()), [dy.to(DEV), dht.to(DEV)])

    def value(s, v):
        z = {n: t.double() + s * v.get(n, 0) for n, t in x.items()}
        h0 = z.pop("initial_state")
        o = scan(**z, softplus=True, h0=h0)
        return ((o["y"] * dy).sum() + (o["ht"] * dht).sum()).item()

    for n, g in zip(d, got):
        v = {n: torch.randn(x[n].shape, dtype=torch.float64,
                            generator=torch.Generator().manual_seed(5))}
        ref = (value(1e-4, v) - value(-1e-4, v)) / 2e-4
        term = (g.cpu().double() * v[n]).abs().sum().item()
        assert abs((g.cpu().double() * v[n]).sum().item() - ref) <= 1e-4 * term, n


def test_extreme_values():
    """delta of -inf keeps the state and passes no gradient; a huge one forgets it; NaN and inf
    stay in their channel and in what follows them."""
    B, T, D, N = 1, 40, 6, 16
    x, _ = make(B, T, D, N, torch.float32)
    x["delta"][0, 10, 0] = float("-inf")
    x["delta"][0, 20, 1] = 1e4
    x["u"][0, 25, 2] = float("nan")
    x["u"][0, 30, 3] = float("inf")
    d = {n: t.to(DEV) for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True)
    y, ht = y.cpu(), ht.cpu()
    ref, mag = reference(x, True, None)
    clean = [0, 1, 4, 5]
    close("y", y[..., clean], ref["y"][..., clean], mag["y"][..., clean], 4 * T + 64)
    close("ht", ht[:, clean], ref["ht"][:, clean], mag["ht"][:, clean], 4 * T + 64)
    assert torch.isfinite(y[0, :25, 2]).all() and torch.isnan(y[0, 25:, 2]).all()
    assert torch.isfinite(y[0, :30, 3]).all() and not torch.isfinite(y[0, 30:, 3]).any()


def test_unused_outputs():
    """Only the final state used, and only y."""
    x, r = make(1, 50, 16, 8, torch.float32)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True)
    dht = r(1, 16, 8)
    names = [n for n in d]
    got = torch.autograd.grad(ht, list(d.values()), dht.to(DEV), retain_graph=True,
                              allow_unused=True)
    ref, mag = reference(x, True, None, torch.zeros(1, 50, 16), dht)
    for n, t in zip(names, got):
        close("d" + n, t, ref["d" + n], mag["d" + n], 4 * 50 + 64 + 66)
    dy = r(1, 50, 16)
    got = torch.autograd.grad(y, list(d.values()), dy.to(DEV))
    ref, mag = reference(x, True, None, dy, torch.zeros(1, 16, 8))
    for n, t in zip(names, got):
        close("d" + n, t, ref["d" + n], mag["d" + n], 4 * 50 + 64 + 66)


def test_empty_calls():
    x, _ = make(2, 0, 24, 16, torch.bfloat16)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True)
    assert y.shape == (2, 0, 24) and torch.equal(ht, d["initial_state"])
    g = torch.autograd.grad(ht, [d["initial_state"], d["A"]], torch.ones_like(ht))
    assert (g[0] == 1).all() and (g[1] == 0).all()
    x, _ = make(0, 5, 24, 16, torch.bfloat16)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True)
    assert y.shape == (0, 5, 24) and ht.shape == (0, 24, 16)
    assert (torch.autograd.grad(y, d["A"], y.detach())[0] == 0).all()


def test_repeatable():
    """The same inputs give the same bits: sums have a fixed order."""
    x, r = make(2, 300, 260, 16, torch.bfloat16)
    dy = r(2, 300, 260).to(torch.bfloat16).to(DEV)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    runs = []
    for _ in range(3):
        y, _ = selective_scan(**d, delta_softplus=True)
        runs.append([y.detach(), *torch.autograd.grad(y, list(d.values()), dy)])
    for run in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], run))


def test_other_stream_and_graph():
    """On a side stream, and captured into a graph that is replayed on new inputs."""
    x, r = make(2, 150, 64, 16, torch.bfloat16)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    dy = r(2, 150, 64).to(torch.bfloat16).to(DEV)

    def step():
        y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True)
        return [y.detach(), ht.detach(), *torch.autograd.grad(y, list(d.values()), dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            d["u"].copy_(torch.randn(2, 150, 64, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        # seed 0 is the first input again (make's first draw), the others are new ones
        assert torch.equal(side[0], out[0]) == (k == 0)


def test_no_second_derivative():
    x, _ = make(1, 20, 8, 4, torch.float32)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, _ = selective_scan(**d, delta_softplus=True)
    g, = torch.autograd.grad(y.sum(), d["u"], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, None), (3, 20, 16, None), (5, 257, 16, None),
                                     (2, 48, 7, None), (4, 24, 20, 4), (2, 18, 64, 3),
                                     (130, 2048, 16, None)])
def test_step(B, D, N, G, dt):
    x, r = make(B, 1, D, N, dt, G=G)
    state = x["initial_state"].to(DEV)
    one = {n: t[:, 0] if n in ("u", "delta", "z", "B", "C") else t for n, t in x.items()}
    del one["initial_state"]
    args = {n: t.to(DEV) for n, t in one.items()}
    y = selective_scan_step(state, **args, delta_softplus=True)
    assert y.dtype == dt
    ref, mag = reference(x, True, None)
    close("y", y[:, None], ref["y"], mag["y"], 68)
    close("state", state, ref["ht"], mag["ht"], 68)


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_step_slots(itype):
    """Rows in slots of a pool, rows without one, and slots that nobody names."""
    B, D, N = 6, 40, 16
    x, r = make(B, 1, D, N, torch.float32)
    pool = r(2, 9, D, N)[1]
    slots = torch.tensor([4, -1, 0, 9, 8, -7], dtype=itype)
    x["initial_state"] = pool[slots.clamp(0, 8).long()].clone()
    ref, mag = reference(x, True, None)
    dev = torch.zeros(9, 2, D, N, device=DEV)[:, 0]   # slots that are not next to each other
    dev.copy_(pool)
    args = {n: t.to(DEV)[:, 0] if n in ("u", "delta", "z", "B", "C") else t.to(DEV)
            for n, t in x.items() if n != "initial_state"}
    y = selective_scan_step(dev, **args, delta_softplus=True, state_indices=slots.to(DEV))
    live = [0, 2, 4]
    close("y", y[live], ref["y"][live, 0], mag["y"][live, 0], 68)
    assert (y[[1, 3, 5]] == 0).all()
    close("state", dev[[4, 0, 8]], ref["ht"][live], mag["ht"][live], 68)
    rest = [1, 2, 3, 5, 6, 7]
    assert torch.equal(dev[rest].cpu(), pool[rest])


def test_steps_equal_the_scan():
    x, _ = make(2, 20, 48, 16, torch.float32)
    d = {n: t.to(DEV) for n, t in x.items()}
    state = d.pop("initial_state").clone()
    ys = []
    for t in range(20):
        ys.append(selective_scan_step(
            state, **{n: v[:, t] if v.dim() == 3 else v for n, v in d.items()},
            delta_softplus=True))
    ref, mag = reference(x, True, None)
    close("y", torch.stack(ys, 1), ref["y"], mag["y"], 4 * 20 + 64)
    close("state", state, ref["ht"], mag["ht"], 4 * 20 + 64)


def test_step_strided_views():
    x, _ = make(3, 1, 40, 13, torch.bfloat16)
    ref, mag = reference(x, True, None)
    state = x["initial_state"].to(DEV)
    args = {}
    for n, t in x.items():
        if n in ("u", "delta", "z", "B", "C"):
            t = t[:, 0].to(DEV)
            args[n] = torch.cat([t, t, t], -1)[:, t.shape[1]:2 * t.shape[1]]
        elif n != "initial_state":
            args[n] = t.to(DEV)
    y = selective_scan_step(state, **args, delta_softplus=True)
    close("y", y[:, None], ref["y"], mag["y"], 68)


def test_empty_step():
    x, _ = make(1, 1, 8, 4, torch.float32)
    args = {n: t[:0, 0].to(DEV) if n in ("u", "delta", "z", "B", "C") else t.to(DEV)
            for n, t in x.items() if n != "initial_state"}
    assert selective_scan_step(torch.zeros(0, 8, 4, device=DEV), **args).shape == (0, 8)


def test_step_of_a_state_that_a_backward_needs():
    """The step counts as an in-place operation on its state: an expression that kept it for its
    backward says so instead of using the new values. States without a counter work as before."""
    x, _ = make(2, 1, 24, 16, torch.float32)
    d = {n: t[:, 0].to(DEV) if n in ("u", "delta", "z", "B", "C") else t.to(DEV)
         for n, t in x.items()}
    pool = d.pop("initial_state")
    w = torch.ones_like(pool).requires_grad_()
    loss, version = (w * pool).sum(), pool._version
    selective_scan_step(pool, **d, delta_softplus=True)
    assert pool._version > version
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():
        state = pool.clone()
        assert state.is_inference()
        want = selective_scan_step(pool, **d, delta_softplus=True)
        assert torch.equal(selective_scan_step(state, **d, delta_softplus=True), want)
        assert torch.equal(state, pool)


def test_empty_batch_of_long_sequences():
    x, _ = make(0, 100, 24, 16, torch.bfloat16)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=True, output_final_state=True)
    assert y.shape == (0, 100, 24) and ht.shape == (0, 24, 16)
    g = torch.autograd.grad([y, ht], list(d.values()), [y.detach(), ht.detach()])
    assert all(t.shape == d[n].shape and (t == 0).all() for n, t in zip(d, g))
