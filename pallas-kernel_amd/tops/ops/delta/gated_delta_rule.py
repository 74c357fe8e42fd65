"""The gated delta rule on the ``tops_gla_delta_*`` kernels."""

from __future__ import annotations

import math
import struct

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from ... import _lib
from ..._lib import call_on, check_device, dtype_code, require
from ..ssm._common import (address, device_table, differentiable, f32, gradients, io_dtype,
                           offsets, refuse_grad, rows, slot_args, strides)

_ARGS = struct.Struct("=39qd13q")
_SIZES = struct.Struct("=8q")
_STEP = struct.Struct("=34qd")
_NO_BWD = (0,) * 13


def _gate(t):
    """g or beta as the kernels read it: bfloat16 or float32, its heads contiguous."""
    if t.dtype is not torch.bfloat16 and t.dtype is not torch.float32:
        t = t.to(torch.float32)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _tokens(t, dt):
    """``rows`` of [B, T, heads, columns]; the kernels step from token to token in 32 bits."""
    t = rows(t, dt)
    return t if t.shape[1] <= 1 or 0 <= t.stride(1) < 1 << 24 else t.contiguous()


_CUS = 256


def _segment(counts, blocks):
    """Chunks in a segment of packed sequences of ``counts`` chunks, with ``blocks`` blocks for the
    heads and columns of each; tops_gla_delta_segment has the rule for equal lengths.

    All segments should run at once, or the last ones wait for a whole one (lengths of 28, 5, 33,
    2, 47, 1, 8 and 9 chunks, 16 heads of 128 x 128: L = 10 has 272 blocks and takes 219 us, 11 has
    256 and 182, 12 190, 17 239, uncut 357). Where the sequences alone are more than half of what
    the CUs hold, their ends differ anyway, and what is long among them is cut by the average (32
    such heads: L = 17 293 us, uncut 381; 40 of 4 chunks and one of 200: 441, uncut 1505; 64 of 6
    and one of 60: 463, uncut 523)."""
    longest = max(counts)
    L = max(-(-sum(counts) * blocks // _CUS), 2, math.isqrt(max(0, longest - 1) // 4) + 1)
    if 2 * len(counts) * blocks <= _CUS:
        while L < longest and sum(-(-n // L) for n in counts) * blocks > _CUS:
            L += max(1, L // 32)
    return L if longest >= 6 and longest >= 2 * L else max(1, longest)


def _columns(K):
    """Columns of a block of the passes: with more than 128 keys 64. (8 heads of
    256 x 256, 128 chunks: 391 us in segments of 16, 469 in those of 8 that 128 columns would give;
    the packed sequences above 310 for 386.)"""
    return 128 if K <= 128 else 64


class _Chunks:
    """The chunks that a call's sequences are cut into, and the segments that these run in."""

    def __init__(self, B, T, cu, dt, HV, K, V, device):
        lib = _lib.load()
        C = lib.tops_gla_delta_chunk(dtype_code(dt))
        self.table = None
        if cu is None:
            per = -(-T // C)
            self.nseq, self.n = B, B * per
            self.L = lib.tops_gla_delta_segment(B, self.n, HV, V * 128 // _columns(K))
            self.nsegs = B * max(1, -(-per // self.L))
            return
        self.nseq = len(cu) - 1
        counts = [-((a - b) // C) for a, b in zip(cu, cu[1:])]
        self.n = sum(counts)
        blocks = HV * -(-V // _columns(K))

        def make():
            L = _segment(counts, blocks)
            chunks, segs, seq = [0], [0], []
            for s, n in enumerate(counts):
                k = max(1, -(-n // L))
                chunks.append(chunks[-1] + n)
                segs.append(segs[-1] + k)
                seq += [s] * k
            return [*cu, *chunks, *segs, *seq], (len(seq), L)

        key = "delta", tuple(cu), C, blocks
        self.table, (self.nsegs, self.L) = device_table(key, make, device)

    def bytes(self, HV, K, V, dt, train, backward):
        return _lib.load().tops_gla_delta_bytes(
            _SIZES.pack(self.nseq, self.n, self.nsegs, HV, K, V, dtype_code(dt), int(train)),
            int(backward))


def _pack(x, h0, o, ht, keep, nkeep, ch, shape, norm, train, scale, bwd=_NO_BWD):
    q, k, v, g, beta = x
    return _ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), address(h0),
        address(o), address(ht), address(ch.table), address(keep), nkeep, ch.nseq, ch.n, ch.nsegs,
        ch.L, *shape,
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *g.stride()[:2], *beta.stride()[:2],
        int(norm), int(train), dtype_code(q.dtype), dtype_code(g.dtype), dtype_code(beta.dtype),
        scale, *bwd)


def _forward(q, k, v, g, beta, h0, scale, norm, want, cu, train):
    dev = check_device(q, k, v, g, beta, h0)
    dt = io_dtype(q, k, v)
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    x = _tokens(q, dt), _tokens(k, dt), _tokens(v, dt), _gate(g), _gate(beta)
    h0 = f32(h0)
    ch = _Chunks(B, T, cu, dt, HV, K, V, dev)
    o = torch.empty(B, T, HV, V, dtype=dt, device=dev)
    ht = torch.empty(ch.nseq, HV, K, V, dtype=torch.float32, device=dev) if want else None
    nkeep = ch.bytes(HV, K, V, dt, train, False)
    keep = torch.empty(nkeep, dtype=torch.uint8, device=dev)
    call_on(dev, "tops_gla_delta_fwd", _pack(x, h0, o, ht, keep, nkeep, ch,
                                             (B, T, H, HV, K, V), norm, train, scale))
    return o if dt is v.dtype else o.to(v.dtype), ht, x, keep, ch


class _GatedDeltaRuleFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, h0, scale, norm, want, cu):
        ctx.set_materialize_grads(False)
        o, ht, x, keep, ch = _forward(q, k, v, g, beta, h0, scale, norm, want, cu, True)
        ctx.save_for_backward(*x, keep)
        ctx.like = [None if t is None else t.dtype for t in (q, k, v, g, beta, h0)]
        ctx.scale, ctx.norm, ctx.ch = scale, norm, ch
        return o, ht

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dht):
        *x, keep = ctx.saved_tensors
        q, k, v, g, beta = x
        dev, dt, ch = q.device, q.dtype, ctx.ch
        B, T, H, K = q.shape
        HV, V = v.shape[2:]
        do = torch.zeros(B, T, HV, V, dtype=dt, device=dev) if do is None else _tokens(do, dt)
        dht = f32(dht)
        new = torch.empty
        dq, dk = new(B, T, H, K, dtype=dt, device=dev), new(B, T, H, K, dtype=dt, device=dev)
        dv = new(B, T, HV, V, dtype=dt, device=dev)
        dg = new(B, T, HV, dtype=g.dtype, device=dev)
        dbeta = new(B, T, HV, dtype=beta.dtype, device=dev)
        dh0 = (None if ctx.like[5] is None
               else new(ch.nseq, HV, K, V, dtype=torch.float32, device=dev))
        nws = ch.bytes(HV, K, V, dt, True, True)
        ws = new(nws, dtype=torch.uint8, device=dev)
        bwd = [do.data_ptr(), *strides(do, 0, 1, 2), *(address(t) for t in (
            dht, dq, dk, dv, dg, dbeta, dh0, ws)), nws]
        call_on(dev, "tops_gla_delta_bwd", _pack(
            x, None, None, None, keep, keep.numel(), ch, (B, T, H, HV, K, V), ctx.norm, True,
            ctx.scale, bwd))
        grads = (dq, dk, dv, dg, dbeta, dh0)
        return (*gradients(grads, ctx.like, ctx.needs_input_grad), None, None, None, None)


def _check_heads(qs, ks, vs, gs, bs, lead):
    """Shapes of q and k [*lead, H, K], v [*lead, HV, V], g and beta [*lead, HV]."""
    n = len(lead)
    if len(vs) != n + 2 or vs[:n] != lead or ks != qs or qs[:n] != lead:
        require(False, f"q and k must be {[*lead, 'H', 'K']}, v {[*lead, 'HV', 'V']}, got "
                       f"{tuple(qs)}, {tuple(ks)} and {tuple(vs)}")
    H, K = qs[n:]
    HV, V = vs[n:]
    if H < 1 or HV < 1 or HV % H or K < 1 or V < 1:
        require(False, f"the value heads must be a multiple of the key heads, and no size 0: got "
                       f"{tuple(qs)} and {tuple(vs)}")
    if K > 256:
        raise NotImplementedError(f"keys of more than 256 columns: {K}")
    if gs != (*lead, HV) or bs != (*lead, HV):
        require(False, f"g and beta must be {(*lead, HV)}, got {tuple(gs)} and {tuple(bs)}")
    return H, HV, K, V


def gated_delta_rule(q, k, v, g, beta, scale=None, initial_state=None, output_final_state=False,
                     cu_seqlens=None, qk_l2norm=False):
    """Gated delta rule over sequences, differentiable in every tensor.

    Per value head, with a state S of K x V::

        S'  = exp(g_t) S_{t-1}
        n_t = beta_t (v_t - S'^T k_t)        # what the key does not hold yet
        S_t = S' + k_t n_t^T
        o_t = scale S_t^T q_t

    Args:
        q, k: ``[B, T, H, K]``, K <= 256.  v: ``[B, T, HV, V]``, HV a multiple of H: value head j
            uses key head ``j // (HV / H)``.
        g: ``[B, T, HV]``, log decays (-inf: the state is forgotten).  beta: ``[B, T, HV]``.
            Keys of about unit length and 0 <= beta <= 2 keep the state bounded.
        scale: of the outputs, ``K ** -0.5`` by default.
        initial_state: ``[sequences, HV, K, V]`` or None (zeros).
        cu_seqlens: offsets of sequences packed into one row (B == 1), from 0 to T, known on the
            host; empty sequences keep their state.
        qk_l2norm: q and k stand for ``x / sqrt(sum(x^2) + 1e-6)`` of each head.

    Inputs may be views with any strides whose last dimension is contiguous (others are copied).
    bfloat16 q, k and v are read and written as they are, and multiplied in bfloat16 with float32
    sums. States are float32, and multiplied as three bfloat16 parts of 24 bits: final states and
    gradients of initial ones are as exact as float32 sums. What o and the other gradients are made
    of is multiplied in two parts of 16 bits: they are rounded once, to their type. Other types of
    q, k and v are computed in float32. g and beta are read in float32 or bfloat16, whatever the
    others' type, and their gradients returned in it: float32 ones beside bfloat16 q, k and v are
    about 1e-5 off.

    An input that is not finite makes the outputs of its token and of all later ones of the sequence
    not finite, for the value heads that it belongs to; one of v does so in its column, and one of q
    at its own token alone. Gradients may then be not finite for all tokens of the sequence, in the
    heads that share the key head. Nothing else changes, to the bit.
    A second derivative raises.

    Returns ``(o, final_state)``: o ``[B, T, HV, V]`` in v's type, final_state ``[sequences, HV, K,
    V]`` float32 with ``output_final_state``, else None.
    """
    if q.dim() != 4:
        require(False, f"q must be [B, T, H, K], got {tuple(q.shape)}")
    B, T = q.shape[:2]
    H, HV, K, V = _check_heads(q.shape, k.shape, v.shape, g.shape, beta.shape, (B, T))
    cu = offsets(cu_seqlens, B, T)
    S = B if cu is None else len(cu) - 1
    if initial_state is not None and initial_state.shape != (S, HV, K, V):
        require(False, f"initial_state must be {(S, HV, K, V)}, got {tuple(initial_state.shape)}")
    scale = K ** -0.5 if scale is None else float(scale)
    if K < 8 or V < 8:   # the kernels read 8 columns at a time: zeros beside them change nothing
        pk, pv = max(0, 8 - K), max(0, 8 - V)
        o, ht = gated_delta_rule(
            F.pad(q, (0, pk)), F.pad(k, (0, pk)), F.pad(v, (0, pv)), g, beta, scale,
            None if initial_state is None else F.pad(initial_state, (0, pv, 0, pk)),
            output_final_state, cu, qk_l2norm)
        return o[..., :V], None if ht is None else ht[..., :K, :V]
    args = (q, k, v, g, beta, initial_state)
    if differentiable(*args):
        return _GatedDeltaRuleFunction.apply(*args, scale, bool(qk_l2norm),
                                             bool(output_final_state), cu)
    return _forward(*args, scale, bool(qk_l2norm), bool(output_final_state), cu, False)[:2]


def gated_delta_rule_step(state, q, k, v, g, beta, scale=None, qk_l2norm=False,
                          state_indices=None):
    """The next token, or the few next ones, of ``gated_delta_rule`` for each row of a serving
    batch; ``state`` is updated in place.

    Args:
        state: float32 ``[slots, HV, K, V]``, each slot contiguous and none on another.
        q, k: ``[B, H, K]``.  v: ``[B, HV, V]``.  g, beta: ``[B, HV]``. Or all of them with T
            tokens, in their order: ``[B, T, H, K]``, ``[B, T, HV, V]``, ``[B, T, HV]``.
        scale, qk_l2norm: as for ``gated_delta_rule``.
        state_indices: int32 or int64 ``[B]`` on the device, the slot of each row (None: row b
            uses slot b). A row whose slot is negative or not below ``slots`` is left out: no
            state changes for it and its o is 0. No slot may be given to two rows.

    Returns o, of v's shape and type.
    """
    refuse_grad("gated_delta_rule_step", state, q, k, v, g, beta)
    qs, vs, ss = q.shape, v.shape, state.shape
    if len(qs) not in (3, 4):
        require(False, f"q must be [B, H, K] or [B, T, H, K], got {tuple(qs)}")
    one = len(qs) == 3
    lead = tuple(qs[:1 if one else 2])
    H, HV, K, V = _check_heads(qs, k.shape, vs, g.shape, beta.shape, lead)
    B, T = lead[0], 1 if one else lead[1]
    st = state.stride()
    if (len(ss) != 4 or ss[1:] != (HV, K, V) or state.dtype is not torch.float32
            or (st[3] != 1 and V > 1) or (st[2] != V and K > 1) or (st[1] != K * V and HV > 1)
            or (st[0] < HV * K * V and ss[0] > 1)):
        require(False, f"state must be float32 [slots, {HV}, {K}, {V}] with contiguous slots that "
                       "do not overlap")
    if state_indices is None and ss[0] < B:
        require(False, f"state holds {ss[0]} slots, the batch {B}")
    idx, idx64 = slot_args(state_indices, B, q)
    dev = check_device(state, q, k, v, g, beta, state_indices)
    dt = io_dtype(q, k, v)
    qq, kk, vv, gg, bb = rows(q, dt), rows(k, dt), rows(v, dt), _gate(g), _gate(beta)
    o = torch.empty(vs, dtype=dt, device=dev)
    a, b, c, d, e = qq.stride(), kk.stride(), vv.stride(), gg.stride(), bb.stride()
    if one:
        a, b, c = (a[0], 0, a[1]), (b[0], 0, b[1]), (c[0], 0, c[1])
        d, e = (d[0], 0), (e[0], 0)
    call_on(dev, "tops_gla_delta_step", _STEP.pack(
        state.data_ptr(), qq.data_ptr(), kk.data_ptr(), vv.data_ptr(), gg.data_ptr(),
        bb.data_ptr(), o.data_ptr(), idx, idx64, ss[0], B, T, H, HV, K, V, st[0], *a[:3], *b[:3],
        *c[:3], *d[:2], *e[:2], 1 if qk_l2norm else 0, dtype_code(dt), dtype_code(gg.dtype),
        dtype_code(bb.dtype), K ** -0.5 if scale is None else scale))
    increment_version(state)   # as torch's own in-place operations do
    return o if dt is v.dtype else o.to(v.dtype)
