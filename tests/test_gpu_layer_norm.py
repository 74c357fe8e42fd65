"""layer_norm against the norm in 64 bits.

Bounds in the 2-norm: half a step of the result's type, and the roundings of float32 sums. A sum of
D terms is one of at most 32 in a row for each thread, 6 levels of lanes and 8 waves: 46, and twice
that for a variance, whose differences are rounded too; dx has two sums on top of y's. The weights'
gradients add rows in runs of at most rows / 16 and 16 partial sums."""

import pytest
import torch

from delta_ref import F64, HALF, ULP32, close, layer_norm as ref_norm
from tops.modules import LayerNorm
from tops.ops.norm import layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FL = torch.bfloat16, torch.float32
SUMS = 3 * 46 + 16


def check(x, w, b, dy, eps=1e-5, to=lambda t: t.to(DEV), f=layer_norm, grow=1.0):
    dt = x.dtype
    d = [None if t is None else to(t).detach().requires_grad_() for t in (x, w, b)]
    y = f(*d, eps=eps)
    assert y.dtype == dt and y.shape == x.shape
    c = [None if t is None else t.to(F64).requires_grad_() for t in (x, w, b)]
    ry = ref_norm(*c, eps=eps)
    out = HALF if dt is BF else ULP32
    close("y", y, ry, out + SUMS * ULP32 * grow)
    names = [n for n, t in zip("xwb", d) if t is not None]
    got = torch.autograd.grad(y, [t for t in d if t is not None], dy.to(DEV))
    ref = torch.autograd.grad(ry, [t for t in c if t is not None], dy.to(F64))
    rows = x.numel() // x.shape[-1]
    for n, t, r, s in zip(names, got, ref, [t for t in (x, w, b) if t is not None]):
        assert t.dtype == s.dtype and t.shape == s.shape
        own = HALF if t.dtype is BF else ULP32
        many = 0 if n == "x" else rows / 16 + 32
        close("d" + n, t, r, own + (2 * SUMS * grow + many) * ULP32, 1e-30 if rows else 1e-12)
    return y


def make(shape, dt, seed=0, offset=0.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)   # noqa: E731
    D = shape[-1]
    return (r(*shape) + offset).to(dt), 1 + 0.2 * r(D), 0.3 * r(D), r(*shape).to(dt)


# features around a run (8, in float32 4), a lane's runs, a wave's (2048) and a block's (8192) rows
@pytest.mark.parametrize("D", [3, 7, 8, 12, 64, 100, 511, 512, 520, 1024, 2047, 2048, 2049, 2056,
                               4100, 8192, 8193, 8200, 16383, 16384])
@pytest.mark.parametrize("dt", [FL, BF])
def test_forward_backward(D, dt):
    check(*make((5, D), dt))


@pytest.mark.parametrize("rows", [1, 3, 4, 1000, 5000])
@pytest.mark.parametrize("dt", [FL, BF])
def test_rows(rows, dt):
    check(*make((rows, 48), dt))


@pytest.mark.parametrize("rows,D", [(3000, 1100), (700, 5000), (600, 9000)])
@pytest.mark.parametrize("dt", [FL, BF])
def test_more_rows_than_blocks(rows, D, dt):
    check(*make((rows, D), dt))


@pytest.mark.parametrize("shape", [(0, 16), (2, 0, 16), (16,), (2, 3, 4, 16)])
def test_shapes(shape):
    check(*make(shape, FL))


@pytest.mark.parametrize("w,b", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("dt", [FL, BF])
def test_without_weight_or_bias(w, b, dt):
    x, ww, bb, dy = make((6, 72), dt)
    check(x, ww if w else None, bb if b else None, dy)


def test_types_of_weights():
    x, w, b, dy = make((6, 72), BF)
    check(x, w.to(BF), b.to(BF), dy)


@pytest.mark.parametrize("dt", [torch.float16, F64])
def test_other_types(dt):
    x, w, b, _ = make((6, 72), FL)
    y = layer_norm(x.to(dt).to(DEV), w.to(DEV), b.to(DEV))
    assert y.dtype == dt
    close("y", y, ref_norm(x.to(dt).to(F64), w.to(F64), b.to(F64)),
          SUMS * ULP32 + torch.finfo(torch.float16).eps / 2)


def test_large_means():
    """A mean of 1000 standard deviations: the differences lose 10 bits of x, no more."""
    check(*make((8, 512), FL, offset=1000.0), grow=1024)


def test_rows_without_variance():
    x, w, b, _ = make((3, 40), FL)
    x[1] = 2.0
    y = layer_norm(x.to(DEV), w.to(DEV), b.to(DEV))
    assert torch.equal(y[1].cpu(), b)
    close("y", y, ref_norm(x.to(F64), w.to(F64), b.to(F64)), SUMS * ULP32)


def test_rows_are_independent():
    x, w, b, _ = make((9, 200), BF)
    y = layer_norm(x.to(DEV), w.to(DEV), b.to(DEV))
    x[4] = torch.inf
    x[5, 3] = torch.nan
    z = layer_norm(x.to(DEV), w.to(DEV), b.to(DEV))
    keep = [0, 1, 2, 3, 6, 7, 8]
    assert torch.equal(y[keep], z[keep]) and z[4:6].isnan().all()


@pytest.mark.parametrize("dt", [FL, BF])
def test_views(dt):
    x, w, b, dy = make((6, 72), dt)
    check(x, w, b, dy, to=lambda t: torch.cat([t, t], -1)[..., t.shape[-1]:].to(DEV)
          if t.dim() > 1 else t.to(DEV))

    def odd(t):   # rows that begin at odd addresses
        if t.dim() == 1:
            return t.to(DEV)
        wide = torch.zeros(t.shape[0], 2 * t.shape[1] + 1, dtype=t.dtype, device=DEV)
        wide[:, 1:1 + t.shape[1]] = t.to(DEV)
        return wide[:, 1:1 + t.shape[1]]

    check(x, w, b, dy, to=odd)
    check(x, w, b, dy, to=lambda t: t.to(DEV).t().contiguous().t() if t.dim() > 1 else t.to(DEV))
    x3, w, b, dy3 = make((4, 5, 24), dt)
    check(x3, w, b, dy3, to=lambda t: t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
          if t.dim() > 2 else t.to(DEV))


def test_expanded_upstream():
    x, w, b, _ = make((6, 72), FL)
    d = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    one = torch.autograd.grad(layer_norm(*d).sum(), d)
    two = torch.autograd.grad(layer_norm(*d), d, torch.ones(6, 72, device=DEV))
    assert all(torch.equal(a, c) for a, c in zip(one, two))


def test_repeats_and_graphs():
    x, w, b, dy = (t.to(DEV) for t in make((3000, 256), BF))
    d = [t.requires_grad_() for t in (x, w, b)]

    def call():
        y = layer_norm(*d)
        return [y.detach(), *torch.autograd.grad(y, d, dy)]

    first = call()
    assert all(torch.equal(a, c) for a, c in zip(first, call()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        with torch.no_grad():
            x.mul_(0.9).add_(0.1 * i)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(want, out)), i


def test_rows_past_2_31_elements():
    rows, D = (1 << 31) // 8192 + 3, 8192
    x = torch.zeros(rows, D, dtype=BF, device=DEV)
    tail = torch.randn(2, D, device=DEV).to(BF)
    x[-2:] = tail
    with torch.no_grad():
        assert torch.equal(layer_norm(x)[-2:], layer_norm(tail))


def test_module():
    m = LayerNorm(72, device=DEV)
    assert [n for n, _ in m.named_parameters()] == ["weight", "bias"]
    x, w, b, dy = make((6, 72), BF)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    close("y", m(x.to(DEV)), ref_norm(*(t.to(F64) for t in (x, w, b))), HALF + SUMS * ULP32)
    plain = LayerNorm(72, elementwise_affine=False, eps=1e-3)
    assert not list(plain.parameters())
    close("y", plain(x.to(DEV)), ref_norm(x.to(F64), eps=1e-3), HALF + SUMS * ULP32)
    half = LayerNorm(72, bias=False)
    assert [n for n, _ in half.named_parameters()] == ["weight"]
