"""Per-head RMS norms of queries and keys and their position rotation, one pass over both, on the
``tops_gla_qk_norm_rope_*`` kernels."""

from __future__ import annotations

import struct

import torch
from torch.autograd.function import once_differentiable

from ... import _lib
from ..._lib import call, check_device, dtype_code, require, stream_of
from ..ssm._common import address, differentiable, f32, io_dtype, rows, strides

_ARGS = struct.Struct("=8q 6q 8q 2q d 2q 6q 4q 2q")


_NO_BWD = (0,) * 14


def rotary_inv_freq(rotary_dim, theta=10000.0, device=None):
    """The usual frequencies ``theta^(-2 i / rotary_dim)``, float64 ``[rotary_dim / 2]``."""
    require(rotary_dim >= 0 and rotary_dim % 2 == 0, "rotary_dim must be even")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    return float(theta) ** (-i / max(1, rotary_dim))


def _pack(x, out, interleaved, eps, bwd=None):
    q, k, qw, kw, freq, pos = x
    B, T, Hq, D = q.shape
    pos_sb = pos64 = 0
    if pos is not None:
        pos64 = 1 if pos.dtype is torch.int64 else 0
        if pos.dim() == 2:
            pos_sb = pos.stride(0)
    return _ARGS.pack(
        q.data_ptr(), k.data_ptr(), address(qw), address(kw), address(freq), address(pos),
        address(out[0]), address(out[1]), B, T, Hq, k.shape[2], D,
        0 if freq is None else 2 * freq.shape[0], *q.stride()[:3], *k.stride()[:3], pos_sb, pos64,
        1 if interleaved else 0, dtype_code(q.dtype), eps, *(bwd or _NO_BWD))


def _forward(q, k, qw, kw, freq, pos, eps, interleaved):
    dev = check_device(q, k, qw, kw, freq, pos)
    dt = io_dtype(q, k)
    x = (rows(q, dt), rows(k, dt), f32(qw), f32(kw), freq, pos)
    qo = torch.empty(q.shape, dtype=dt, device=dev)
    ko = torch.empty(k.shape, dtype=dt, device=dev)
    call("tops_gla_qk_norm_rope_fwd", _pack(x, (qo, ko), interleaved, eps), stream_of(dev))
    return qo if dt is q.dtype else qo.to(q.dtype), ko if dt is k.dtype else ko.to(k.dtype), x


class _QkNormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, freq, pos, eps, interleaved):
        ctx.set_materialize_grads(False)
        qo, ko, x = _forward(q, k, qw, kw, freq, pos, eps, interleaved)
        ctx.save_for_backward(*x)
        ctx.meta = eps, interleaved
        ctx.like = [None if t is None else t.dtype for t in (q, k, qw, kw)]
        return qo, ko

    @staticmethod
    @once_differentiable
    def backward(ctx, dqo, dko):
        x = ctx.saved_tensors
        q, k, qw, kw = x[:4]
        eps, interleaved = ctx.meta
        dev, dt = q.device, q.dtype
        D = q.shape[-1]
        g = [torch.zeros(t.shape, dtype=dt, device=dev) if d is None else rows(d, dt)
             for t, d in ((q, dqo), (k, dko))]
        dq, dk = (torch.empty(t.shape, dtype=dt, device=dev) for t in (q, k))
        need = ctx.needs_input_grad
        dqw = torch.empty(D, dtype=torch.float32, device=dev) if need[2] else None
        dkw = torch.empty(D, dtype=torch.float32, device=dev) if need[3] else None
        nws, ws = 0, None
        if need[2] or need[3]:
            nws = int(_lib.load().tops_gla_qk_norm_rope_ws_bytes(q.shape[0] * q.shape[1], D))
            ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        bwd = [address(g[0]), address(g[1]), *strides(g[0], 0, 1, 2), *strides(g[1], 0, 1, 2),
               *(address(t) for t in (dq, dk, dqw, dkw, ws)), nws]
        call("tops_gla_qk_norm_rope_bwd", _pack(x, (None, None), interleaved, eps, bwd),
             stream_of(dev))
        return (*(t if t is None or not n else t.to(like)
                  for t, n, like in zip((dq, dk, dqw, dkw), need, ctx.like)),
                None, None, None, None)


def qk_norm_rope(q, k, q_weight=None, k_weight=None, inv_freq=None, positions=None, *, eps=1e-6,
                 interleaved=False):
    """RMS norm of every head of q and k, then the rotation by the token's position::

        n = x * rsqrt(mean(x^2) + eps) * weight        (over the head's D columns)
        n[i], n[j] <- n[i] cos a - n[j] sin a, n[j] cos a + n[i] sin a,   a = position inv_freq[p]

    for the pairs p of the first ``2 len(inv_freq)`` columns: (p, p + len(inv_freq)), or
    (2 p, 2 p + 1) with ``interleaved``. The other columns are normed only. Computed in float32
    and rounded once; the angles are formed in 64 bits, which far positions need.

    Args:
        q, k: ``[B, T, Hq, D]`` and ``[B, T, Hk, D]``, D <= 512; views of a fused projection
            are read in place (any strides with the last dimension contiguous).
        q_weight, k_weight: ``[D]`` or None.
        inv_freq: float64 ``[R / 2]``, R <= D (``rotary_inv_freq``), or None for no rotation.
        positions: int32 or int64 ``[B, T]`` or ``[T]``; None: 0 .. T - 1 in every row.

    Differentiable in q, k and the weights. Returns ``(q', k')`` in the inputs' types, contiguous.
    """
    qs, ks = q.shape, k.shape
    if (len(qs) != 4 or len(ks) != 4 or qs[0] != ks[0] or qs[1] != ks[1] or qs[3] != ks[3]
            or not 1 <= qs[3] <= 512):
        require(False, f"q and k must be [B, T, heads, D] with one D <= 512, got "
                       f"{tuple(qs)} and {tuple(ks)}")
    B, T, _, D = qs
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and w.shape != (D,):
            require(False, f"{name} must be {(D,)}, got {tuple(w.shape)}")
    if inv_freq is not None:
        if inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > D or inv_freq.dtype is not torch.float64:
            require(False, f"inv_freq must be float64 [R / 2] with R <= {D}, got "
                           f"{inv_freq.dtype} {tuple(inv_freq.shape)}")
        if not inv_freq.is_contiguous():
            inv_freq = inv_freq.contiguous()
    if positions is not None:
        if (positions.dtype not in (torch.int32, torch.int64)
                or positions.shape not in ((B, T), (T,))):
            require(False, f"positions must be int32 or int64 {(B, T)} or {(T,)}, got "
                           f"{positions.dtype} {tuple(positions.shape)}")
        if positions.shape[-1] > 1 and positions.stride(-1) != 1:
            positions = positions.contiguous()
    args = (q, k, q_weight, k_weight)
    if differentiable(*args):
        return _QkNormRopeFunction.apply(*args, inv_freq, positions, float(eps), bool(interleaved))
    return _forward(*args, inv_freq, positions, float(eps), bool(interleaved))[:2]
