"""Causal depthwise convolution with a carried window, on the ``tops_gla_causal_conv_*``
kernels."""

from __future__ import annotations

import struct

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from ... import _lib
from ..._lib import call, check_device, dtype_code, require, stream_of
from ._common import (address, device_table, differentiable, gradients, io_dtype, offsets,
                      refuse_grad, rows, slot_args, strides)

_ARGS = struct.Struct("=27q")
_STEP = struct.Struct("=16q")

def _cu_tensor(cu, device):
    """The offsets as a device int32 array."""
    return None if cu is None else device_table(tuple(cu), lambda: (cu, None), device)[0]


def _silu(activation):
    if activation not in (None, "silu", "swish"):
        require(False, f"activation must be None, 'silu' or 'swish', got {activation!r}")
    return activation is not None


def _contiguous(t, dt):
    if t is None or (t.dtype is dt and t.is_contiguous()):
        return t
    return t.to(dt).contiguous()


def _check_weight(weight, bias, D, W):
    if weight.shape not in ((D, W), (D, 1, W)) or not 1 <= W <= 8 or D < 1:
        require(False, f"weight must be [{D}, W] or [{D}, 1, W] with W <= 8, got "
                       f"{tuple(weight.shape)}")
    if bias is not None and bias.shape != (D,):
        require(False, f"bias must be {(D,)}, got {tuple(bias.shape)}")


def _pack(x, y, fin, cu_t, nseq, silu, bwd=None):
    xx, w, b, init = x
    B, T, D = xx.shape
    return _ARGS.pack(address(xx), address(w), address(b), address(init), address(y),
                      address(fin), address(cu_t), nseq, B, T, D, w.shape[1], *strides(xx, 0, 1),
                      int(silu), dtype_code(xx.dtype), dtype_code(w.dtype), *(bwd or [0] * 10))


def _forward(x, weight, bias, init, silu, want, cu):
    dev = check_device(x, weight, bias, init)
    dt = io_dtype(x)
    B, T, D = x.shape
    W = weight.shape[-1]
    wt = io_dtype(weight, bias)
    a = (rows(x, dt), _contiguous(weight if weight.dim() == 2 else weight.reshape(D, W), wt),
         _contiguous(bias, wt), _contiguous(init, dt))
    nseq = B if cu is None else len(cu) - 1
    cu_t = _cu_tensor(cu, dev)
    y = torch.empty(B, T, D, dtype=dt, device=dev)
    fin = torch.empty(nseq, W, D, dtype=dt, device=dev) if want else None
    call("tops_gla_causal_conv_fwd", _pack(a, y, fin, cu_t, nseq, silu), stream_of(dev))
    if dt is not x.dtype:
        y, fin = y.to(x.dtype), None if fin is None else fin.to(x.dtype)
    return y, fin, a, cu_t


class _CausalConvFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, init, silu, want, cu):
        ctx.set_materialize_grads(False)
        y, fin, a, cu_t = _forward(x, weight, bias, init, silu, want, cu)
        ctx.save_for_backward(*a, cu_t)
        ctx.like = [None if t is None else t.dtype for t in (x, weight, bias, init)]
        ctx.wshape = weight.shape
        ctx.silu, ctx.nseq = silu, x.shape[0] if cu is None else len(cu) - 1
        return y, fin

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfin):
        x, w, b, init, cu_t = ctx.saved_tensors
        dev, dt = x.device, x.dtype
        B, T, D = x.shape
        W = w.shape[1]
        dy = torch.zeros(B, T, D, dtype=dt, device=dev) if dy is None else rows(dy, dt)
        dfin = _contiguous(dfin, dt)
        dx = torch.empty(B, T, D, dtype=dt, device=dev)
        dinit = None if init is None else torch.empty(ctx.nseq, W, D, dtype=dt, device=dev)
        dw = db = ws = None
        nws = 0
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dw = torch.empty(ctx.wshape, dtype=w.dtype, device=dev)
            db = None if b is None else torch.empty(D, dtype=w.dtype, device=dev)
            nws = int(_lib.load().tops_gla_causal_conv_bwd_ws_bytes(B * T, D, W))
            ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        bwd = [*(address(t) for t in (dy, dfin, dx, dinit, dw, db, ws)), nws, *strides(dy, 0, 1)]
        call("tops_gla_causal_conv_bwd", _pack((x, w, b, init), None, None, cu_t, ctx.nseq,
                                               ctx.silu, bwd), stream_of(dev))
        return (*gradients((dx, dw, db, dinit), ctx.like, ctx.needs_input_grad), None, None,
                None)


def causal_conv1d(x, weight, bias=None, activation=None, initial_state=None,
                  output_final_state=False, cu_seqlens=None):
    """Causal depthwise convolution over time, differentiable in every tensor::

        y_t[d] = act(sum_{j < W} weight[d, j] x_{t - W + 1 + j}[d] + bias[d])

    The rows before a sequence's first token come from ``initial_state`` (zeros without one), so
    that a prompt can be run piece by piece: ``final_state`` of a piece is the ``initial_state``
    of the next, and the ``state`` of ``causal_conv1d_step``. Its layout is the cache of
    ``ShortConvolution``.

    Args:
        x: ``[B, T, D]``, any strides with the last dimension contiguous (others are copied).
        weight: ``[D, W]`` or ``[D, 1, W]``, W <= 8.  bias: ``[D]`` or None.
        activation: None, "silu" or "swish".
        initial_state: ``[sequences, W, D]``, the last W inputs before each sequence (the first
            of them is outside every window).
        cu_seqlens: offsets of sequences packed into one row (B == 1), from 0 to T, known on the
            host; empty sequences keep their state.

    Returns ``(y, final_state)`` in x's type; final_state ``[sequences, W, D]`` with
    ``output_final_state``, else None.
    """
    if x.dim() != 3:
        require(False, f"x must be [B, T, D], got {tuple(x.shape)}")
    B, T, D = x.shape
    W = weight.shape[-1]
    _check_weight(weight, bias, D, W)
    silu = _silu(activation)
    cu = offsets(cu_seqlens, B, T)
    S = B if cu is None else len(cu) - 1
    if initial_state is not None and initial_state.shape != (S, W, D):
        require(False, f"initial_state must be {(S, W, D)}, got {tuple(initial_state.shape)}")
    args = (x, weight, bias, initial_state)
    if differentiable(*args):
        return _CausalConvFunction.apply(*args, silu, bool(output_final_state), cu)
    return _forward(*args, silu, bool(output_final_state), cu)[:2]


def causal_conv1d_step(x, state, weight, bias=None, activation=None, state_indices=None):
    """One token of ``causal_conv1d`` for each row of a serving batch: ``state`` moves up a row
    and takes x, in place.

    Args:
        x: ``[B, D]``.
        state: ``[slots, W, D]`` of x's type, each slot contiguous and none on another.
        weight, bias, activation: as for ``causal_conv1d``.
        state_indices: as for ``selective_scan_step``.

    Returns y ``[B, D]`` in x's type.
    """
    refuse_grad("causal_conv1d_step", x, state, weight, bias)
    shape, ss, dtype = x.shape, state.shape, x.dtype
    if len(shape) != 2:
        require(False, f"x must be [B, D], got {tuple(shape)}")
    B, D = shape
    W = weight.shape[-1]
    _check_weight(weight, bias, D, W)
    silu = _silu(activation)
    st = state.stride()
    if (len(ss) != 3 or ss[1] != W or ss[2] != D or state.dtype is not dtype
            or (st[2] != 1 and D > 1) or (st[1] != D and W > 1)
            or (st[0] < W * D and ss[0] > 1)):
        require(False, f"state must be {dtype} [slots, {W}, {D}] with contiguous slots that do "
                       "not overlap")
    if state_indices is None and ss[0] < B:
        require(False, f"state holds {ss[0]} slots, the batch {B}")
    idx, idx64 = slot_args(state_indices, B, x)
    dev = check_device(x, state, weight, bias, state_indices)
    dt = dtype_code(dtype)
    wt = io_dtype(weight, bias)
    xx = rows(x, dtype)
    ww, bb = _contiguous(weight, wt), _contiguous(bias, wt)
    y = torch.empty(shape, dtype=dtype, device=dev)
    call("tops_gla_causal_conv_step", _STEP.pack(
        xx.data_ptr(), state.data_ptr(), ww.data_ptr(), address(bb), y.data_ptr(), idx, idx64,
        ss[0], B, D, W, st[0], xx.stride(0), int(silu), dt, dtype_code(wt)), stream_of(dev))
    increment_version(state)   # as torch's own in-place operations do
    return y
