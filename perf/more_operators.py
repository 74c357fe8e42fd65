"""Performance cases of the gated delta rule and of the layer norm.

Three operators, each through the public entry points:

* ``delta``     : ``gated_delta_rule``, prompts (fixed length or packed, states carried in and
                  out) and training (forward + backward);
* ``delta_step``: ``gated_delta_rule_step``, the next token, or the few next ones, of a serving
                  batch, states updated in place;
* ``norm``      : ``layer_norm``, prompts, decoding and training (forward + backward).

A case is a dict of plain values; ``lengths`` (text) gives the packed sequences' lengths.
"""

import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = 64
L2_EPS = 1e-6
EPS = 1e-5

own = False   # False: the plain forms; True: the framework's entry points


def listed():
    return [
        # one user's short prompt: latency
        dict(name="delta_prompt_short", kind="delta", B=1, T=200, H=8, HV=8, K=64, V=64,
             dtype="bf16", train=False, carry=False, l2norm=True, lengths=""),
        # prompts of different lengths packed into one row, states carried on, a key head for two
        # value heads
        dict(name="delta_prefill_packed", kind="delta", B=1, T=8192, H=8, HV=16, K=128, V=128,
             dtype="bf16", train=False, carry=True, l2norm=True,
             lengths="1733,290,2049,77,3001,512,1,529"),
        # one long prompt: nothing but its heads runs in parallel along the recurrence
        dict(name="delta_prefill_long", kind="delta", B=1, T=16384, H=16, HV=16, K=128, V=128,
             dtype="bf16", train=False, carry=True, l2norm=True, lengths=""),
        # a training step's delta rule
        dict(name="delta_train", kind="delta", B=2, T=4096, H=16, HV=16, K=128, V=128,
             dtype="bf16", train=True, carry=False, l2norm=True, lengths=""),
        # training on a document cut into pieces, shared key heads, values wider than keys
        dict(name="delta_train_grouped", kind="delta", B=1, T=5000, H=4, HV=8, K=64, V=128,
             dtype="bf16", train=True, carry=True, l2norm=True, lengths=""),
        # float32 training at sizes that divide by nothing, keys normed by the caller
        dict(name="delta_train_float32", kind="delta", B=3, T=1001, H=4, HV=4, K=100, V=72,
             dtype="f32", train=True, carry=True, l2norm=False, lengths=""),
        # one user's next token
        dict(name="delta_step_one", kind="delta_step", B=1, T=1, H=8, HV=16, K=128, V=128,
             slots=0, dtype="bf16", l2norm=True),
        # the next token of a serving batch, its states in a pool of slots
        dict(name="delta_step_batch", kind="delta_step", B=128, T=1, H=16, HV=16, K=128, V=128,
             slots=160, dtype="bf16", l2norm=True),
        # four accepted drafted tokens of each of a small batch
        dict(name="delta_step_tokens", kind="delta_step", B=16, T=4, H=16, HV=16, K=128, V=128,
             slots=24, dtype="bf16", l2norm=True),
        # the norm of a serving batch's next token
        dict(name="norm_decode", kind="norm", rows=64, D=2048, dtype="bf16", train=False),
        # a training step's norm
        dict(name="norm_train", kind="norm", rows=32768, D=2048, dtype="bf16", train=True),
        # float32 training at an odd size
        dict(name="norm_train_float32", kind="norm", rows=3003, D=1001, dtype="f32", train=True),
    ]


LARGEST = 2 * 4096 * 16 * 128 * 128   # tokens x state elements of the listed training case


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _documents(rng, total):
    """Text of the lengths of 2 to 20 documents of `total` tokens."""
    n = min(total, _log(rng, 2, 20))
    parts = [rng.lognormvariate(0.0, 1.2) for _ in range(n)]
    lens = [max(1, int(total * p / sum(parts))) for p in parts]
    return ",".join(str(x) for x in lens)


def _heads(rng):
    H = rng.choice([1, 2, 4, 8, 16])
    HV = H * rng.choice([g for g in (1, 1, 2, 4) if H * g <= 32])
    return dict(H=H, HV=HV, K=rng.choice([64, 128, 128, 128, 96, 80, 100]),
                V=rng.choice([64, 128, 128, 128, 96, 72, 200, 256]))


def draw(rng):
    """A case of the listed ones' ranges."""
    what = rng.choice(["step", "step", "tokens", "prompt", "prompt", "packed", "train", "train",
                       "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if what.startswith("norm"):
        D = _log(rng, 64, 8192)
        D = D if rng.random() < 0.3 else max(8, D // 8 * 8)
        most = 32768 * 2048 // D // (1 if dtype == "bf16" else 2)
        return dict(kind="norm", rows=_log(rng, 1, most), D=D, dtype=dtype,
                    train=what == "norm_train")
    heads = _heads(rng)
    size = heads["HV"] * heads["K"] * heads["V"]
    if what in ("step", "tokens"):
        B = _log(rng, 1, min(128, 128 * 16 * 128 * 128 // size))
        return dict(kind="delta_step", B=B, T=1 if what == "step" else rng.choice([2, 3, 4, 5, 8]),
                    **heads, slots=rng.choice([0, B + 7]), dtype=dtype, l2norm=rng.random() < 0.8)
    # float32 products run on matrix units of a sixteenth of the rate
    most = LARGEST // size // (1 if what == "train" else 2) // (1 if dtype == "bf16" else 8)
    tokens = _log(rng, 64, max(65, min(16384, most)))
    lengths = _documents(rng, tokens) if what == "packed" else ""
    B = 1 if what == "packed" else rng.choice([1, 2, 4, 8])
    T = sum(int(n) for n in lengths.split(",")) if lengths else max(1, tokens // B)
    return dict(kind="delta", B=B, T=T, **heads, dtype=dtype, train=what == "train",
                carry=what == "packed" or rng.random() < 0.5, l2norm=rng.random() < 0.8,
                lengths=lengths)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _cu(case):
    """Offsets of the packed sequences, or None."""
    if not case.get("lengths"):
        return None
    cu = [0]
    for n in case["lengths"].split(","):
        cu.append(cu[-1] + int(n))
    return cu


def _sequences(case):
    cu = _cu(case)
    return case["B"] if cu is None else len(cu) - 1


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def mk(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=DEV)

    leaf = (lambda t: t.detach().requires_grad_(bool(case.get("train"))))   # noqa: E731
    if case["kind"] == "norm":
        rows, D = case["rows"], case["D"]
        x = {"x": (0.3 * mk(1, D) + mk(rows, D)).to(dt), "weight": 1 + 0.1 * mk(D),
             "bias": 0.1 * mk(D)}
        st = dict(case=case, x={n: leaf(t) for n, t in x.items()})
        if case["train"]:
            st["dy"] = mk(rows, D).to(dt)
        return st
    B, T, H, HV, K, V = (case[n] for n in ("B", "T", "H", "HV", "K", "V"))
    # the convolution's output holds queries, keys and values side by side
    silu = torch.nn.functional.silu
    nq = H * K
    mixed = silu(mk(B, T, 2 * nq + HV * V))
    if not case["l2norm"]:   # queries and keys of about unit length
        mixed[..., :2 * nq] *= 1.7 * K ** -0.5
    mixed = mixed.to(dt)
    x = {"q": mixed[..., :nq].unflatten(-1, (H, K)),
         "k": mixed[..., nq:2 * nq].unflatten(-1, (H, K)),
         "v": mixed[..., 2 * nq:].unflatten(-1, (HV, V))}
    # decay rates of 1 to 16 and steps of 0.001 to 0.1, as training begins with, changed by the
    # token; written strengths between 0 and 1. In float32, or in the type of the rest where their
    # gradients are wanted
    dtg = dt if case.get("train") else torch.float32
    rate, step = 1 + 15 * rand(HV), torch.exp(math.log(1e-3) + math.log(100.0) * rand(HV))
    pre = mk(B, T, HV) + step + torch.log(-torch.expm1(-step))
    x["g"] = (-rate * torch.nn.functional.softplus(pre)).to(dtg)
    x["beta"] = torch.sigmoid(mk(B, T, HV)).to(dtg)
    if case["kind"] == "delta_step":
        slots, idx = B, None
        if case["slots"]:
            slots = case["slots"]
            order = torch.randperm(slots, generator=gen, device=DEV)
            idx = order[:B].to(torch.int32)
        return dict(case=case, x=x, idx=idx, state=mk(slots, HV, K, V) * K ** -0.5)
    S = _sequences(case)
    if case["carry"]:
        x["initial_state"] = mk(S, HV, K, V) * K ** -0.5
    st = dict(case=case, x={n: leaf(t) for n, t in x.items()}, cu=_cu(case))
    if case["train"]:
        st["do"] = mk(B, T, HV, V).to(dt)
        st["dht"] = mk(S, HV, K, V) if case["carry"] else None
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state)
    with torch.no_grad():
        return {"delta": _delta_plain, "delta_step": _step_plain, "norm": _norm_plain}[kind](state)


def _own(state):
    """The calls of a user's program."""
    if os.path.join(ROOT, "pallas-kernel_amd") not in sys.path:
        sys.path.insert(0, os.path.join(ROOT, "pallas-kernel_amd"))
    import tops.ops.delta as delta
    import tops.ops.norm as norm

    case, x = state["case"], state["x"]
    if case["kind"] == "delta_step":
        q, k, v, g, beta = (x[n] for n in ("q", "k", "v", "g", "beta"))
        if case["T"] == 1:
            q, k, v, g, beta = (t[:, 0] for t in (q, k, v, g, beta))
        with torch.no_grad():
            o = delta.gated_delta_rule_step(state["state"], q, k, v, g, beta,
                                            qk_l2norm=case["l2norm"], state_indices=state["idx"])
        return {"o": o, "state": state["state"]}
    train = bool(case["train"])
    with torch.set_grad_enabled(train):
        if case["kind"] == "norm":
            outs = [norm.layer_norm(x["x"], x["weight"], x["bias"], eps=EPS)]
            names, grads = ["y"], [state.get("dy")]
        else:
            keep = case["carry"]
            o, ht = delta.gated_delta_rule(
                x["q"], x["k"], x["v"], x["g"], x["beta"], qk_l2norm=case["l2norm"],
                initial_state=x.get("initial_state"), output_final_state=keep,
                cu_seqlens=state["cu"])
            names, outs = ["o", "ht"][:1 + keep], [o, ht][:1 + keep]
            grads = [state.get("do"), state.get("dht")][:1 + keep]
    res = {n: o.detach() for n, o in zip(names, outs)}
    if train:
        res["grads"] = dict(zip(x, torch.autograd.grad(outs, list(x.values()), grads)))
    return res


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _norm_plain(state):
    dt = DTYPES[state["case"]["dtype"]]
    x, w, b = (state["x"][n].float() for n in ("x", "weight", "bias"))
    xc = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    n = xc * r
    out = {"y": (n * w + b).to(dt)}
    if state["case"]["train"]:
        dy = state["dy"].float()
        dn = dy * w
        dx = r * (dn - dn.mean(-1, keepdim=True) - n * (dn * n).mean(-1, keepdim=True))
        out["grads"] = {"x": dx.to(dt), "weight": (dy * n).sum(0), "bias": dy.sum(0)}
    return out


def _unit(x):
    """(rows of unit length, what they were multiplied by)."""
    r = torch.rsqrt((x * x).sum(-1, keepdim=True) + L2_EPS)
    return x * r, r


def _step_plain(state):
    case = state["case"]
    x = {n: t.float() for n, t in state["x"].items()}
    group = case["HV"] // case["H"]
    q, k = x["q"], x["k"]
    if case["l2norm"]:
        q, k = _unit(q)[0], _unit(k)[0]
    q, k = (t.repeat_interleave(group, 2) * s for t, s in ((q, case["K"] ** -0.5), (k, 1)))
    idx = slice(None) if state["idx"] is None else state["idx"].long()
    h = state["state"][idx]
    o = []
    for t in range(case["T"]):
        h = h * torch.exp(x["g"][:, t])[..., None, None]
        n = (x["v"][:, t] - (h * k[:, t, ..., None]).sum(-2)) * x["beta"][:, t, :, None]
        h = h + k[:, t, ..., None] * n[..., None, :]
        o.append((h * q[:, t, ..., None]).sum(-2))
    state["state"][idx] = h
    o = torch.stack(o, 1).to(DTYPES[case["dtype"]])
    return {"o": o[:, 0] if case["T"] == 1 else o, "state": state["state"]}


def _chunk_rows(case):
    """The tokens of all sequences in chunks that no sequence shares, [chunks, CHUNK] with the
    number of tokens where a chunk ends early, and the chunks of each sequence."""
    cu = _cu(case)
    if cu is None:
        cu = [b * case["T"] for b in range(case["B"] + 1)]
    tok, first, count = cu[-1], [], []
    ends, starts = [], []
    for a, b in zip(cu, cu[1:]):
        first.append(len(starts))
        count.append(-(-(b - a) // CHUNK))
        starts += range(a, b, CHUNK)
        ends += [b] * count[-1]
    rows = torch.tensor(starts)[:, None] + torch.arange(CHUNK)
    rows = torch.where(rows < torch.tensor(ends)[:, None], rows, tok).to(DEV)
    return rows, tok, first, count


def _delta_plain(state):
    """Chunk by chunk: within one, the new values solve a unit triangular system, whose inverse is
    a product of powers; from one to the next goes the state."""
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]
    H, HV, K, V = (case[n] for n in ("H", "HV", "K", "V"))
    group, scale = HV // H, K ** -0.5
    rows, tok, first, count = _chunk_rows(case)

    def cut(t):   # [B, T, heads, ...] -> [chunks, heads, CHUNK, ...] in float32
        t = t.float().flatten(0, 1)
        return torch.cat([t, torch.zeros_like(t[:1])])[rows].transpose(1, 2)

    def back(t):   # and back
        out = t.new_zeros(tok + 1, *t.shape[1:2], *t.shape[3:])
        out[rows] = t.transpose(1, 2)
        return out[:tok].unflatten(0, (case["B"], case["T"]))

    x = state["x"]
    q, k, v, beta = cut(x["q"]), cut(x["k"]), cut(x["v"]), cut(x["beta"])[..., None]
    if case["l2norm"]:
        (q, rq), (k, rk) = _unit(q), _unit(k)
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    G = cut(x["g"]).double().cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=DEV).tril()
    D = torch.exp(torch.where(lower, G[..., None] - G[..., None, :], -torch.inf)).float()
    eg, el = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None]
    last = eg[..., -1:, :]
    kt = k.transpose(-1, -2).contiguous()
    A = (beta * (k @ kt) * D).tril(-1)
    Ti, p = torch.eye(CHUNK, device=DEV) - A, A
    for _ in range(5):   # (1 + A)^-1 = (1 - A)(1 + A^2)(1 + A^4) ...
        p = p @ p
        Ti = Ti + Ti @ p
    P = scale * (q @ kt) * D
    W, U = Ti @ (beta * eg * k), Ti @ (beta * v)

    seqs = range(len(count))
    steps = [[s for s in seqs if n < count[s]] for n in range(max(count))]
    at = [([first[s] + n for s in act], act) for n, act in enumerate(steps)]
    cur = torch.zeros(len(count), HV, K, V, device=DEV)
    if case["carry"]:
        cur = x["initial_state"].float().clone()
    S, N = torch.empty(len(rows), HV, K, V, device=DEV), torch.empty_like(U)
    kel = (k * el).transpose(-1, -2).contiguous()
    for c, act in at:
        h = cur[act]
        S[c] = h
        n = U[c] - W[c] @ h
        N[c] = n
        cur[act] = last[c] * h + kel[c] @ n
    qs = q @ S
    out = {"o": back(scale * eg * qs + P @ N).to(dt)}
    if case["carry"]:
        out["ht"] = cur
    if not case["train"]:
        return out

    do = cut(state["do"])
    dcur = state["dht"].clone() if case["carry"] else torch.zeros_like(cur)
    dS, Y = torch.empty_like(S), torch.empty_like(N)
    dn0 = P.transpose(-1, -2).contiguous() @ do
    ds0 = (scale * eg * q).transpose(-1, -2).contiguous() @ do
    kb = (beta * eg * k).transpose(-1, -2).contiguous()
    Tt, kg = Ti.transpose(-1, -2).contiguous(), k * el
    for c, act in reversed(at):
        d = dcur[act]
        dS[c] = d
        y = Tt[c] @ (dn0[c] + kg[c] @ d)
        Y[c] = y
        dcur[act] = last[c] * d + ds0[c] - kb[c] @ y
    Nt, St = N.transpose(-1, -2).contiguous(), S.transpose(-1, -2).contiguous()
    dP, dA = (do @ Nt) * D, -(Y @ Nt).tril(-1) * D
    dq = scale * (eg * (do @ St) + dP @ k)
    z = dA @ k - eg * (Y @ St)
    dkl = el * (N @ dS.transpose(-1, -2).contiguous())
    dkw = dkl + scale * dP.transpose(-1, -2).contiguous() @ q
    dkw = dkw + (beta * dA).transpose(-1, -2).contiguous() @ k
    dG = (q * dq + k * (beta * z - dkw)).sum(-1).double()
    dG[..., -1] += (k * dkl).sum((-1, -2)) + (last * S * dS).sum((-1, -2))
    dg = dG.flip(-1).cumsum(-1).flip(-1).float()
    dk = beta * z + dkw
    dq, dk = (t.unflatten(1, (H, group)).sum(2) for t in (dq, dk))
    if case["l2norm"]:
        q, k = q[:, ::group], k[:, ::group]
        dq = rq * (dq - q * (q * dq).sum(-1, keepdim=True))
        dk = rk * (dk - k * (k * dk).sum(-1, keepdim=True))
        k = k.repeat_interleave(group, 1)
    grads = {"q": back(dq).to(dt), "k": back(dk).to(dt), "v": back(beta * Y).to(dt),
             "g": back(dg).to(dt), "beta": back((k * z).sum(-1) + (v * Y).sum(-1)).to(dt)}
    if case["carry"]:
        grads["initial_state"] = dcur
    out["grads"] = grads
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "norm":
        n, D = case["rows"] * case["D"], case["D"]
        if not case["train"]:
            return {"bytes": 2 * n * es + 8 * D, "flops": 7 * n}
        return {"bytes": 4 * n * es + 16 * D, "flops": 20 * n}
    tok = case["B"] * case["T"]
    H, HV, K, V = (case[n] for n in ("H", "HV", "K", "V"))
    kv, vv, states = 2 * tok * H * K * es, tok * HV * V * es, 4 * HV * K * V
    if case["kind"] == "delta_step":
        return {"bytes": kv + 2 * vv + 8 * tok * HV + 2 * case["B"] * states,
                "flops": tok * HV * 7 * K * V}
    carried = _sequences(case) * states if case["carry"] else 0
    if not case["train"]:
        return {"bytes": kv + 2 * vv + 8 * tok * HV + 2 * carried, "flops": tok * HV * 7 * K * V}
    return {"bytes": 2 * kv + 4 * vv + 4 * tok * HV * es + 4 * carried,
            "flops": tok * HV * 22 * K * V}


# ---------------------------------------------------------------------------
# the same values in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    x = {n: t.detach().double() for n, t in st["x"].items()}
    if case["kind"] == "norm":
        return _norm64(case, st, x)
    heads = case["HV"] // case["H"]
    leaves = {n: x[n].requires_grad_(bool(case.get("train"))) for n in ("q", "k")}
    with torch.set_grad_enabled(bool(case.get("train"))):
        rows = {}
        for n, t in leaves.items():   # one row for each value head
            if case["l2norm"]:
                t = t / torch.sqrt(t.square().sum(-1, keepdim=True) + L2_EPS)
            rows[n] = t[:, :, :, None].expand(-1, -1, -1, heads, -1).flatten(2, 3)
    q, k = rows["q"].detach() / math.sqrt(case["K"]), rows["k"].detach()
    if case["kind"] == "delta_step":
        idx = torch.arange(case["B"], device=DEV) if st["idx"] is None else st["idx"].long()
        pool = st["state"].double()
        o, pool[idx], _ = _tokens64(q, k, x["v"], x["g"], x["beta"], pool[idx])
        return {"o": o[:, 0] if case["T"] == 1 else o, "state": pool}
    cu = st["cu"]
    pieces = [slice(None)] if cu is None else [slice(a, b) for a, b in zip(cu, cu[1:])]
    outs, ends, gs, dh = [], [], [], []
    for i, at in enumerate(pieces):
        part = [t[:, at] for t in (q, k, x["v"], x["g"], x["beta"])]
        h = torch.zeros(case["B"], case["HV"], case["K"], case["V"], dtype=torch.float64,
                        device=DEV)
        if case["carry"]:
            h = x["initial_state"] if cu is None else x["initial_state"][i:i + 1]
        do = dht = None
        if case["train"]:
            do, dht = st["do"][:, at].double(), torch.zeros_like(h)
            if case["carry"]:
                dht = st["dht"].double() if cu is None else st["dht"][i:i + 1].double()
        o, h, g = _tokens64(*part, h, do, dht)
        outs.append(o)
        ends.append(h)
        if case["train"]:
            gs.append(g[:-1])
            dh.append(g[-1])
    out = {"o": torch.cat(outs, 1)}
    if case["carry"]:
        out["ht"] = torch.cat(ends)
    if case["train"]:
        dq, dk, dv, dg, dbeta = (torch.cat(ts, 1) for ts in zip(*gs))
        grads = dict(zip(("q", "k"), torch.autograd.grad(
            [rows["q"], rows["k"]], [leaves["q"], leaves["k"]],
            [dq / math.sqrt(case["K"]), dk])), v=dv, g=dg, beta=dbeta)
        if case["carry"]:
            grads["initial_state"] = torch.cat(dh)
        out["grads"] = grads
    return out


def _tokens64(q, k, v, g, beta, h, do=None, dht=None):
    """The recurrence token by token, and with do its adjoint in the reverse order:
    (o, final state, gradients of the inputs or None)."""
    o, kept = torch.empty_like(v), []
    for t in range(q.shape[1]):
        kept.append(h if do is not None else None)
        h = torch.exp(g[:, t])[:, :, None, None] * h
        e = v[:, t] - torch.einsum("bhkv,bhk->bhv", h, k[:, t])
        h = h + torch.einsum("bhk,bhv->bhkv", k[:, t], beta[:, t, :, None] * e)
        o[:, t] = torch.einsum("bhkv,bhk->bhv", h, q[:, t])
    if do is None:
        return o, h, None
    dq, dk, dv, dg, db = (torch.empty_like(t) for t in (q, k, v, g, beta))
    end, d = h, dht
    for t in reversed(range(q.shape[1])):
        a, b = torch.exp(g[:, t])[:, :, None, None], beta[:, t, :, None]
        faded = a * kept[t]
        e = v[:, t] - torch.einsum("bhkv,bhk->bhv", faded, k[:, t])
        after = faded + torch.einsum("bhk,bhv->bhkv", k[:, t], b * e)
        dq[:, t] = torch.einsum("bhkv,bhv->bhk", after, do[:, t])
        d = d + torch.einsum("bhk,bhv->bhkv", q[:, t], do[:, t])
        dw = torch.einsum("bhkv,bhk->bhv", d, k[:, t])   # of what is written
        db[:, t] = (dw * e).sum(-1)
        dv[:, t] = b * dw
        dk[:, t] = (torch.einsum("bhkv,bhv->bhk", d, b * e)
                    - torch.einsum("bhkv,bhv->bhk", faded, b * dw))
        d = d - torch.einsum("bhk,bhv->bhkv", k[:, t], b * dw)
        dg[:, t] = (d * faded).sum((-1, -2))
        d = a * d
        kept[t] = None
    return o, end, (dq, dk, dv, dg, db, d)


def _norm64(case, st, x):
    leaves = {n: t.requires_grad_(bool(case["train"])) for n, t in x.items()}
    with torch.set_grad_enabled(bool(case["train"])):
        var, mean = torch.var_mean(leaves["x"], -1, keepdim=True, correction=0)
        y = (leaves["x"] - mean) / torch.sqrt(var + EPS) * leaves["weight"] + leaves["bias"]
    out = {"y": y.detach()}
    if case["train"]:
        out["grads"] = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()),
                                                            st["dy"].double())))
    return out
