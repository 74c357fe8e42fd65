"""Host helpers of the selective state space operators."""

from __future__ import annotations

import threading

import torch

from ..._lib import require, stream_of, to_list

_IO = (torch.float32, torch.bfloat16)


def io_dtype(*tensors):
    """The type the kernel computes such tensors in: bfloat16 where all are, else float32."""
    for t in tensors:
        if t is not None and t.dtype is not torch.bfloat16:
            return torch.float32
    return torch.bfloat16


def rows(t, dt):
    """t in type dt with its last dimension contiguous (a view where it already is)."""
    if t is None or (t.dtype is dt and t.stride(-1) == 1):
        return t
    t = t.to(dt)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def f32(t):
    """A small parameter or a state as the kernels read it: float32, contiguous."""
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.to(torch.float32).contiguous()


def differentiable(*tensors):
    """Whether a call has to go through autograd (forward-mode differentiation included, which
    the functions then refuse)."""
    if torch.autograd.forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def refuse_grad(name, *tensors):
    if torch.is_grad_enabled() and differentiable(*tensors):
        raise RuntimeError(f"{name} updates its state in place and has no gradient: call it under "
                           "torch.no_grad()")


def offsets(cu_seqlens, B, T):
    """Packed sequences' token offsets as a list (empty sequences allowed), or None."""
    if cu_seqlens is None:
        return None
    cu = to_list(cu_seqlens)
    if B != 1:
        require(False, f"cu_seqlens requires B == 1, got B={B}")
    if (len(cu) < 2 or cu[0] != 0 or cu[-1] != T
            or any(b < a for a, b in zip(cu, cu[1:]))):
        require(False, f"cu_seqlens must go from 0 to T={T} without decreasing: {cu}")
    return cu


_tables: dict = {}
_held: list = []
_tables_lock = threading.Lock()


def device_table(key, make, device):
    """``make()`` -> (int32 values, anything else) with the values as a device tensor, kept by its
    key, device and stream: one stream writes, reads and frees a table, in this order. A table
    that a graph captures is kept for good, as the graph's replays read it."""
    key = (key, device.index, stream_of(device).value)
    capturing = torch.cuda.is_current_stream_capturing()
    with _tables_lock:
        hit = _tables.get(key)
        if hit is None and capturing:
            # a capture runs on its own stream, and cannot upload a table of its own
            hit = next((v for k, v in _tables.items() if k[:2] == key[:2]), None)
            if hit is None:
                raise RuntimeError("packed sequences in a graph capture: run the call once with "
                                   "the same cu_seqlens before the capture")
        if hit is None:
            values, rest = make()
            if len(_tables) > 64:
                _tables.clear()
            # pinned, so that the copy is one of the stream's own and nothing waits for it
            table = torch.tensor(values, dtype=torch.int32, pin_memory=True)
            hit = _tables[key] = (table.to(device, non_blocking=True), rest)
        if capturing and not any(h is hit for h in _held):
            _held.append(hit)
    return hit


def slot_args(idx, batch, device_of):
    """(address, whether int64) of the state slots of a batch."""
    if idx is None:
        return 0, 0
    if idx.dtype not in (torch.int32, torch.int64) or idx.shape != (batch,):
        require(False, f"state_indices must be int32 or int64 of shape {(batch,)}, got "
                       f"{idx.dtype} {tuple(idx.shape)}")
    require(batch <= 1 or idx.stride(0) == 1, "state_indices must be contiguous")
    return idx.data_ptr(), int(idx.dtype == torch.int64)


def gradients(grads, like, need):
    """The gradients in the types of their inputs, None where none is wanted."""
    return [None if g is None or not n else g if g.dtype is dt else g.to(dt)
            for g, dt, n in zip(grads, like, need)]


def address(t):
    return 0 if t is None else t.data_ptr()


def strides(t, *dims):
    if t is None:
        return (0,) * len(dims)
    s = t.stride()
    return [s[d] for d in dims]
