"""Plain 64-bit forms of the gated delta rule and of the layer norm, differentiable by torch, and
how far the kernels' results may be from them.

A result of a bfloat16 call may be off by one half step (2^-8) for each operand on its way that is
rounded to bfloat16, and for itself, in the 2-norm over the tensor; one of float32 products by the
roundings of their sums. States go through operands of two bfloat16 parts, each 2^-18 off."""

import torch

F64 = torch.float64
HALF = 2.0 ** -8          # half a step of bfloat16
ULP32 = 2.0 ** -24        # and of float32


def ranges(B, T, cu):
    if cu is None:
        return [(b, 0, T) for b in range(B)]
    return [(0, a, b) for a, b in zip(cu, cu[1:])]


def unit(x):
    return x / torch.sqrt(x.square().sum(-1, keepdim=True) + 1e-6)


def delta(q, k, v, g, beta, h0=None, scale=None, cu=None, l2norm=False):
    """(o, final states) token by token, all tensors float64."""
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    scale = K ** -0.5 if scale is None else scale
    if l2norm:
        q, k = unit(q), unit(k)
    q, k = (t.repeat_interleave(HV // H, 2) for t in (q, k))
    rows, ends = {}, []
    for s, (b, t0, t1) in enumerate(ranges(B, T, cu)):
        h = torch.zeros(HV, K, V, dtype=F64) if h0 is None else h0[s]
        for t in range(t0, t1):
            h = torch.exp(g[b, t])[:, None, None] * h
            n = beta[b, t, :, None] * (v[b, t] - (h * k[b, t, :, :, None]).sum(1))
            h = h + k[b, t, :, :, None] * n[:, None]
            rows[b, t] = scale * (h * q[b, t, :, :, None]).sum(1)
        ends.append(h)
    o = [torch.stack([rows[b, t] for t in range(T)]) if T else v.new_zeros(0, HV, V)
         for b in range(B)]
    o = torch.stack(o) if B else v.new_zeros(0, T, HV, V)
    return o, torch.stack(ends) if ends else v.new_zeros(0, HV, K, V)


def layer_norm(x, w=None, b=None, eps=1e-5):
    c = x - x.mean(-1, keepdim=True)
    y = c / torch.sqrt(c.square().mean(-1, keepdim=True) + eps)
    y = y if w is None else y * w
    return y if b is None else y + b


def sum_roundings(K, tokens):
    """Roundings of the float32 sums of a result: over the keys, over a chunk's 64 tokens (three
    products one after another), and one a chunk where the states go on."""
    return K + 3 * 64 + tokens // 32 + 32


# operands rounded to bfloat16 on the way to a result, and its own rounding:
#   o: the state, the written values, the scores, o;  dq: the written values (in the scores'
#   gradient), the state, the scores' gradient, dq;  dk: the written values, the right side's
#   gradient, both states, the two gradients of scores, dk;  dv: the right side's gradient, dv;
#   dbeta: that, the state, the written values, the system's gradient, dbeta;  dg: all of them, as
#   a difference of sums that are no more than twice its terms
ROUNDED = {"o": 4, "q": 4, "k": 7, "v": 2, "beta": 5, "g": 16}


def bound(name, dt, K, tokens):
    f32 = sum_roundings(K, tokens) * ULP32
    if name in ("ht", "initial_state"):
        # the state, the inverse, the right side and the values, each in two parts, twice over (the
        # gradient goes through the scores too)
        return f32 if dt is torch.float32 else f32 + 10 * 2.0 ** -18
    if dt is torch.float32:   # a gradient is made of results of the forward
        return f32 * (1 if name == "o" else 3 if name != "g" else 6)
    return ROUNDED[name] * HALF


def close(name, got, want, tol, floor=1e-30):
    got, want = got.detach().cpu().to(F64), want.detach()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), name
    err, size = (got - want).norm().item(), want.norm().item()
    assert err <= tol * size + floor, f"{name}: {err / max(size, floor):.3g} off, {tol:.3g} allowed"
