"""Layer norm on the ``tops_gla_layer_norm_*`` kernels."""

from __future__ import annotations

import struct

import torch
from torch.autograd.function import once_differentiable

from ... import _lib
from ..._lib import call_on, check_device, dtype_code, require
from ..ssm._common import address, differentiable, f32, gradients, io_dtype

_ARGS = struct.Struct("=9qd7q")


def _rows(t, dt, D):
    """(t in type dt, the distance of its rows): a view where its rows lie evenly."""
    t = t if t.dtype is dt else t.to(dt)
    if t.dim() == 2 and (t.stride(1) == 1 or D == 1):
        return t, t.stride(0)
    t = t.reshape(-1, D)
    t = t if t.stride(1) == 1 or D == 1 else t.contiguous()
    return t, t.stride(0)


def _forward(x, weight, bias, eps, keep):
    dev = check_device(x, weight, bias)
    dt = io_dtype(x)
    D = x.shape[-1]
    xx, st = _rows(x, dt, D)
    w, b = f32(weight), f32(bias)
    y = torch.empty(x.shape, dtype=dt, device=dev)
    n = xx.shape[0]
    stats = torch.empty(n, 2, dtype=torch.float32, device=dev) if keep else None
    call_on(dev, "tops_gla_layer_norm_fwd", _ARGS.pack(
        xx.data_ptr(), address(w), address(b), y.data_ptr(), address(stats), n, D, st,
        dtype_code(dt), eps, *(0,) * 7))
    return y if dt is x.dtype else y.to(x.dtype), xx, w, stats


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, xx, w, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(xx, w, stats)
        ctx.like = [None if t is None else t.dtype for t in (x, weight, bias)]
        ctx.shape = x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, stats = ctx.saved_tensors
        dev, dt = x.device, x.dtype
        D = ctx.shape[-1]
        dd, dy_st = _rows(dy, dt, D)
        n = x.shape[0]
        dx = torch.empty(ctx.shape, dtype=dt, device=dev)
        new = torch.empty
        dw = new(D, dtype=torch.float32, device=dev) if ctx.needs_input_grad[1] else None
        db = new(D, dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        ws, nws = None, 0
        if dw is not None or db is not None:
            nws = int(_lib.load().tops_gla_layer_norm_ws_bytes(n, D, dtype_code(dt)))
            ws = new(nws, dtype=torch.uint8, device=dev)
        call_on(dev, "tops_gla_layer_norm_bwd", _ARGS.pack(
            x.data_ptr(), address(w), 0, 0, stats.data_ptr(), n, D, x.stride(0), dtype_code(dt),
            0.0, dd.data_ptr(), dy_st, dx.data_ptr(), address(dw), address(db), address(ws), nws))
        return (*gradients((dx, dw, db), ctx.like, ctx.needs_input_grad), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension, differentiable in every tensor::

        y = (x - mean(x)) / sqrt(mean((x - mean(x))^2) + eps) * weight + bias

    Args:
        x: ``[..., D]``, D <= 16384. Rows that lie evenly, as those of a slice of columns do, are
            read where they are, others are copied.
        weight, bias: ``[D]`` or None (ones, zeros), read in float32.
        eps: at least 0.

    Means, squares and the gradients of weight and bias are float32 inside, bfloat16 rows are read
    and written as they are, other types in float32. The gradients are of a fixed order of sums.
    Returns y in x's type.
    """
    if x.dim() < 1 or x.shape[-1] < 1:
        require(False, f"x must be [..., D] with D >= 1, got {tuple(x.shape)}")
    D = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (D,):
            require(False, f"{name} must be {(D,)}, got {tuple(t.shape)}")
    if not eps >= 0:
        require(False, f"eps must be at least 0, got {eps}")
    if differentiable(x, weight, bias):
        return _LayerNormFunction.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]
