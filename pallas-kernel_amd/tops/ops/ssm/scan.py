"""Selective state space scan on the ``tops_gla_selective_scan_*`` kernels."""

from __future__ import annotations

import struct

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from ... import _lib
from ..._lib import call, check_device, dtype_code, require, stream_of
from ._common import (address, device_table, differentiable, f32, gradients, io_dtype, offsets,
                      refuse_grad, rows, slot_args, strides)

_ARGS = struct.Struct("=53q")
_STEP = struct.Struct("=27q")
_NO_BWD = (0,) * 15
_NONE = (0,) * 4   # the strides of a tensor that is not there


class _Pieces:
    """How the sequences of a call are cut into pieces that run in parallel."""

    def __init__(self, B, T, D, N, G, cu, device):
        lib = _lib.load()
        chunk = lib.tops_gla_selective_scan_chunk(N)
        # packed sequences differ in length: the longest ones are cut however many there are
        self.piece = lib.tops_gla_selective_scan_piece(B * T, B if cu is None else 1, D, N, G)
        self.table = None
        if cu is None:
            per = max(1, -(-T // self.piece))
            self.nseq, self.nsegs = B, B * per
            self.chunks, self.multi = B * -(-T // chunk), self.nsegs > B
            return
        self.nseq = len(cu) - 1

        def make():
            segs, first, c0, multi = [], [], 0, False
            for s, (a, b) in enumerate(zip(cu, cu[1:])):
                n = max(1, -(-(b - a) // self.piece))
                multi |= n > 1
                first.append(len(segs) // 8)
                for i in range(n):
                    t0 = a + i * self.piece
                    segs += [s, t0, min(b, t0 + self.piece), i, n, c0 + i * self.piece // chunk,
                             0, 0]
                c0 += -(-(b - a) // chunk)
            for s, i in enumerate(first):
                segs[8 * s + 6] = i
            return segs, (len(segs) // 8, c0, multi)

        self.table, (self.nsegs, self.chunks, self.multi) = device_table(
            (tuple(cu), self.piece, chunk), make, device)


def _pad(N):
    return 8 if N <= 8 else 16 if N <= 16 else 32 if N <= 32 else 64


def _groups(t, N):
    """B or C as [B, T, G, N]."""
    return t if t.dim() == 4 else t.unsqueeze(2)


def _pack(x, y, ht, chunk_h, ws, bc, pc, shape, softplus, dt, bwd=_NO_BWD):
    Bt, T, D, N, G = shape
    u, delta, A, B, C, Dskip, z, bias, h0 = x
    us, ds, zs, bs, cs = (_NONE if t is None else t.stride() for t in (u, delta, z, B, C))
    ph = pd = 0
    if ws is not None:
        ph = ws.data_ptr()
        pd = ph + 4 * pc.nsegs * _pad(N) * D
    return _ARGS.pack(
        address(u), address(delta), address(z), address(B), address(C), address(A),
        address(Dskip), address(bias), address(h0), address(y), address(ht), address(chunk_h),
        ph, pd, address(bc), address(pc.table),
        pc.nsegs, pc.nseq, pc.piece, Bt, T, D, N, G,
        us[0], us[1], ds[0], ds[1], zs[0], zs[1], *bs[:3], *cs[:3], int(softplus), dtype_code(dt),
        *bwd)


def _piece_states(pc, D, N, dev):
    """Workspace of the pieces' own contributions, [pieces][NP + 1][D] in two parts, where a
    sequence has several pieces."""
    if not pc.multi:
        return None
    return torch.empty(pc.nsegs * (_pad(N) + 1) * D, dtype=torch.float32, device=dev)


def _forward(u, delta, A, B, C, D, z, bias, h0, softplus, want_ht, cu, keep):
    """(y, ht, what the kernel read, chunk states, pieces)."""
    dev = check_device(u, delta, A, B, C, D, z, bias, h0)
    dt = io_dtype(u, delta, B, C, z)
    Bt, T, Dn = u.shape
    N = A.shape[1]
    x = (rows(u, dt), rows(delta, dt), f32(A), rows(_groups(B, N), dt), rows(_groups(C, N), dt),
         f32(D), rows(z, dt), f32(bias), f32(h0))
    G = x[3].shape[2]
    pc = _Pieces(Bt, T, Dn, N, G, cu, dev)
    y = torch.empty(Bt, T, Dn, dtype=dt, device=dev)
    ht = torch.empty(pc.nseq, Dn, N, dtype=torch.float32, device=dev) if want_ht else None
    chunk_h = (torch.empty(pc.chunks, _pad(N), Dn, dtype=torch.float32, device=dev)
               if keep else None)
    ws = _piece_states(pc, Dn, N, dev)
    bc = torch.empty(((Bt * T * G + 1) * 2 + Dn) * _pad(N), dtype=torch.float32, device=dev)
    call("tops_gla_selective_scan_fwd",
         _pack(x, y, ht, chunk_h, ws, bc, pc, (Bt, T, Dn, N, G), softplus, dt), stream_of(dev))
    return y if dt is u.dtype else y.to(u.dtype), ht, x, chunk_h, bc, pc


class _SelectiveScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, h0, softplus, want_ht, cu):
        ctx.set_materialize_grads(False)
        y, ht, x, chunk_h, bc, pc = _forward(u, delta, A, B, C, D, z, bias, h0, softplus, want_ht,
                                             cu, True)
        ctx.save_for_backward(*x[:3], *x[5:8], chunk_h, bc)
        ctx.G, ctx.bshape = x[3].shape[2], B.shape
        ctx.like = [None if t is None else t.dtype for t in (u, delta, A, B, C, D, z, bias, h0)]
        ctx.softplus, ctx.pc = softplus, pc
        return y, ht

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dht):
        u, delta, A, D, z, bias, chunk_h, bc = ctx.saved_tensors
        x = u, delta, A, None, None, D, z, bias, None
        pc, dev, dt = ctx.pc, u.device, u.dtype
        Bt, T, Dn = u.shape
        N, G = A.shape[1], ctx.G
        dy = torch.zeros(Bt, T, Dn, dtype=dt, device=dev) if dy is None else rows(dy, dt)
        dht = f32(dht)

        new, f = torch.empty, torch.float32
        du = new(Bt, T, Dn, dtype=dt, device=dev)
        ddelta = new(Bt, T, Dn, dtype=dt, device=dev)
        dz = None if z is None else new(Bt, T, Dn, dtype=dt, device=dev)
        dB, dC = new(ctx.bshape, dtype=dt, device=dev), new(ctx.bshape, dtype=dt, device=dev)
        dA = new(Dn, N, dtype=f, device=dev)
        dD = None if D is None else new(Dn, dtype=f, device=dev)
        dbias = None if bias is None else new(Dn, dtype=f, device=dev)
        dh0 = None if ctx.like[8] is None else new(pc.nseq, Dn, N, dtype=f, device=dev)
        nws = int(_lib.load().tops_gla_selective_scan_bwd_ws_bytes(Bt * T, pc.nsegs, Dn, N, G))
        ws, ps = new(nws, dtype=torch.uint8, device=dev), _piece_states(pc, Dn, N, dev)
        bwd = [address(dy), *strides(dy, 0, 1), *(address(t) for t in (
            dht, du, ddelta, dz, dB, dC, dA, dD, dbias, dh0, ws)), nws]
        call("tops_gla_selective_scan_bwd",
             _pack(x, None, None, chunk_h, ps, bc, pc,
                   (Bt, T, Dn, N, G), ctx.softplus, dt, bwd), stream_of(dev))
        grads = (du, ddelta, dA, dB, dC, dD, dz, dbias, dh0)
        return (*gradients(grads, ctx.like, ctx.needs_input_grad), None, None, None)


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False,
                   initial_state=None, output_final_state=False, cu_seqlens=None):
    """Selective state space scan, differentiable in every tensor.

    Per channel d with its states n (``delta'`` = ``delta + delta_bias``, its softplus with
    ``delta_softplus``)::

        h_t[n] = exp(delta'_t A[d, n]) h_{t-1}[n] + delta'_t u_t B_t[n]
        y_t    = (sum_n C_t[n] h_t[n] + D[d] u_t) * silu(z_t)

    Args:
        u, delta, z: ``[B, T, D]`` (z optional: the output gate).
        A: ``[D, N]``, N <= 64 (-inf: a state that any ``delta' > 0`` forgets, and that
            ``delta' = 0`` keeps).  B, C: ``[B, T, N]``, or ``[B, T, G, N]`` for G groups of
            D / G consecutive channels each.  D, delta_bias: ``[D]`` or None.
        initial_state: ``[sequences, D, N]`` or None (zeros).
        cu_seqlens: offsets of sequences packed into one row (B == 1), from 0 to T, known on the
            host; empty sequences keep their state.

    Inputs may be views with any strides whose last dimension is contiguous (others are copied).
    bfloat16 tensors are read and written as they are, other types in float32; states, sums and
    the gradients of A, D, delta_bias and the state are float32 inside.

    Returns ``(y, final_state)``: y ``[B, T, D]`` in u's type, final_state ``[sequences, D, N]``
    float32 with ``output_final_state``, else None.
    """
    if u.dim() != 3:
        require(False, f"u must be [B, T, D], got {tuple(u.shape)}")
    Bt, T, Dn = u.shape
    if A.dim() != 2 or A.shape[0] != Dn or not 1 <= A.shape[1] <= 64:
        require(False, f"A must be [{Dn}, N] with 1 <= N <= 64, got {tuple(A.shape)}")
    N = A.shape[1]
    for name, t in (("delta", delta), ("z", z)):
        if t is not None and t.shape != u.shape:
            require(False, f"{name} must be {(Bt, T, Dn)}, got {tuple(t.shape)}")
    for name, t in (("B", B), ("C", C)):
        if (t.dim() not in (3, 4) or t.shape[:2] != u.shape[:2] or t.shape[-1] != N
                or (t.dim() == 4 and (t.shape[2] < 1 or Dn % t.shape[2]))):
            require(False, f"{name} must be [{Bt}, {T}, {N}] or [{Bt}, {T}, G, {N}] with G "
                           f"dividing {Dn}, got {tuple(t.shape)}")
    require(B.shape == C.shape, "B and C must have the same shape")
    require(Dn > 0, "D must be positive")
    for name, t in (("D", D), ("delta_bias", delta_bias)):
        if t is not None and t.shape != (Dn,):
            require(False, f"{name} must be {(Dn,)}, got {tuple(t.shape)}")
    cu = offsets(cu_seqlens, Bt, T)
    S = Bt if cu is None else len(cu) - 1
    if initial_state is not None and initial_state.shape != (S, Dn, N):
        require(False, f"initial_state must be {(S, Dn, N)}, got {tuple(initial_state.shape)}")
    args = (u, delta, A, B, C, D, z, delta_bias, initial_state)
    if differentiable(*args):
        return _SelectiveScanFunction.apply(*args, bool(delta_softplus), bool(output_final_state),
                                            cu)
    return _forward(*args, bool(delta_softplus), bool(output_final_state), cu, False)[:2]


def selective_scan_step(state, u, delta, A, B, C, D=None, z=None, delta_bias=None,
                        delta_softplus=False, state_indices=None):
    """One token of ``selective_scan`` for each row of a serving batch; ``state`` is updated in
    place.

    Args:
        state: float32 ``[slots, D, N]``, each slot contiguous and none on another.
        u, delta, z: ``[B, D]``.  A, D, delta_bias: as for ``selective_scan``.
        B, C: ``[B, N]`` or ``[B, G, N]``.
        state_indices: int32 or int64 ``[B]`` on the device, the slot of each row (None: row b
            uses slot b). A row whose slot is negative or not below ``slots`` is left out: no
            state changes for it and its y is 0. No slot may be given to two rows.

    Returns y ``[B, D]`` in u's type.
    """
    refuse_grad("selective_scan_step", state, u, delta, A, B, C, D, z, delta_bias)
    ushape, ashape, bshape, ss = u.shape, A.shape, B.shape, state.shape
    if len(ushape) != 2 or len(ashape) != 2:
        require(False, f"u must be [B, D], A [D, N], got {tuple(ushape)} and {tuple(ashape)}")
    Bt, Dn = ushape
    N = ashape[1]
    if ashape[0] != Dn or not 1 <= N <= 64 or Dn < 1:
        require(False, f"A must be [{Dn}, N] with 1 <= N <= 64, got {tuple(ashape)}")
    if delta.shape != ushape or (z is not None and z.shape != ushape):
        require(False, f"delta and z must be {(Bt, Dn)}")
    G = bshape[1] if len(bshape) == 3 else 1
    if (bshape != C.shape or len(bshape) not in (2, 3) or bshape[0] != Bt or bshape[-1] != N
            or G < 1 or Dn % G):
        require(False, f"B and C must be [{Bt}, {N}] or [{Bt}, G, {N}] with G dividing {Dn}, got "
                       f"{tuple(bshape)} and {tuple(C.shape)}")
    if ((D is not None and D.shape != (Dn,))
            or (delta_bias is not None and delta_bias.shape != (Dn,))):
        require(False, f"D and delta_bias must be {(Dn,)}")
    st = state.stride()
    if (len(ss) != 3 or ss[1] != Dn or ss[2] != N or state.dtype is not torch.float32
            or (st[2] != 1 and N > 1) or (st[1] != N and Dn > 1)
            or (st[0] < Dn * N and ss[0] > 1)):
        require(False, f"state must be float32 [slots, {Dn}, {N}] with contiguous slots that do "
                       "not overlap")
    if state_indices is None and ss[0] < Bt:
        require(False, f"state holds {ss[0]} slots, the batch {Bt}")
    idx, idx64 = slot_args(state_indices, Bt, u)
    dev = check_device(state, u, delta, A, B, C, D, z, delta_bias, state_indices)
    dt = io_dtype(u, delta, B, C, z)
    uu, dd, bb, cc, zz = rows(u, dt), rows(delta, dt), rows(B, dt), rows(C, dt), rows(z, dt)
    aa, sk, bias = f32(A), f32(D), f32(delta_bias)
    y = torch.empty(ushape, dtype=dt, device=dev)
    bs, cs = bb.stride(), cc.stride()
    call("tops_gla_selective_scan_step", _STEP.pack(
        state.data_ptr(), uu.data_ptr(), dd.data_ptr(), address(zz), bb.data_ptr(), cc.data_ptr(),
        aa.data_ptr(), address(sk), address(bias), y.data_ptr(), idx, idx64, ss[0], Bt, Dn, N, G,
        st[0], uu.stride(0), dd.stride(0), 0 if zz is None else zz.stride(0), bs[0],
        bs[1] if G > 1 else 0, cs[0], cs[1] if G > 1 else 0, 1 if delta_softplus else 0,
        dtype_code(dt)), stream_of(dev))
    increment_version(state)   # as torch's own in-place operations do
    return y if dt is u.dtype else y.to(u.dtype)
