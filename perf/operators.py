"""Performance cases of the selective state space operators and of the rotated, normed queries.

Five operators, each through the public entry points:

* ``scan``     : ``selective_scan``, prompts (fixed length or packed, states carried in and out)
                 and training (forward + backward);
* ``scan_step``: ``selective_scan_step``, a serving batch's next token, states updated in place;
* ``conv``     : ``causal_conv1d``, prompts and training;
* ``conv_step``: ``causal_conv1d_step``, the next token, windows updated in place;
* ``qk``       : ``qk_norm_rope``, the norms of queries and keys for each head with the position
                 rotation, for prompts, training and decoding.

A case is a dict of plain values; ``lengths`` (text) gives the packed sequences' lengths.
"""

import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
THETA = 10000.0

own = False   # False: the plain forms; True: the framework's entry points


def listed():
    return [
        # one user's next token
        dict(name="scan_step_one", kind="scan_step", B=1, D=2048, N=16, slots=0, dtype="bf16"),
        # the next token of a serving batch, its states in a pool of slots
        dict(name="scan_step_batch", kind="scan_step", B=128, D=4096, N=16, slots=160,
             dtype="bf16"),
        # pieces of prompts of different lengths packed into one row, states carried on
        dict(name="scan_prefill_packed", kind="scan", B=1, T=8192, D=2048, N=16, dtype="bf16",
             train=False, carry=True, lengths="1733,290,2049,77,3001,512,1,529"),
        # a training step's scan
        dict(name="scan_train", kind="scan", B=2, T=4096, D=4096, N=16, dtype="bf16", train=True,
             carry=False, lengths=""),
        # float32 training over a long document cut into pieces, sizes that divide by nothing
        dict(name="scan_train_float32", kind="scan", B=3, T=1001, D=1000, N=12, dtype="f32",
             train=True, carry=True, lengths=""),
        # the convolution before the packed prompts' scan
        dict(name="conv_prefill_packed", kind="conv", B=1, T=8192, D=2048, W=4, dtype="bf16",
             train=False, carry=True, bias=True, silu=True,
             lengths="1733,290,2049,77,3001,512,1,529"),
        # a training step's convolution
        dict(name="conv_train", kind="conv", B=4, T=8192, D=4096, W=4, dtype="bf16", train=True,
             carry=False, bias=True, silu=True, lengths=""),
        # the convolution of one user's next token
        dict(name="conv_step_one", kind="conv_step", B=1, D=2048, W=4, bias=True, silu=True,
             slots=0, dtype="bf16"),
        # the convolution of a serving batch's next token
        dict(name="conv_step_batch", kind="conv_step", B=128, D=4096, W=4, bias=True, silu=True,
             slots=160, dtype="bf16"),
        # queries and keys of a serving batch's next token, far positions
        dict(name="qk_decode", kind="qk", B=64, T=1, Hq=16, Hk=4, D=128, R=128, dtype="bf16",
             train=False, interleaved=False, far=True),
        # queries and keys of a long prompt, views of the fused projection, half of a head rotated
        dict(name="qk_prefill", kind="qk", B=1, T=16384, Hq=16, Hk=4, D=128, R=64, dtype="bf16",
             train=False, interleaved=False, far=False),
        # a training step's queries and keys
        dict(name="qk_train", kind="qk", B=4, T=8192, Hq=16, Hk=16, D=128, R=128, dtype="bf16",
             train=True, interleaved=False, far=False),
    ]


LARGEST = 2 * 4096 * 4096 * 16   # states of the largest listed scan, tokens x channels x size


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _documents(rng, total):
    """Text of the lengths of 2 to 20 documents of `total` tokens."""
    n = min(total, _log(rng, 2, 20))
    parts = [rng.lognormvariate(0.0, 1.2) for _ in range(n)]
    lens = [max(1, int(total * p / sum(parts))) for p in parts]
    return ",".join(str(x) for x in lens)


def _channels(rng, hi=4096):
    """Channels: mostly whole 16-byte rows, some of them odd."""
    d = _log(rng, 128, hi)
    return d if rng.random() < 0.2 else max(8, d // 8 * 8)


def draw(rng):
    """A case of the listed ones' ranges."""
    what = rng.choice(["scan_step", "prompt", "prompt", "packed", "train", "train", "conv",
                       "conv_packed", "conv_train", "conv_step", "qk", "qk_train", "qk_decode"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if what == "scan_step":
        B = _log(rng, 1, 128)
        return dict(kind="scan_step", B=B, D=_channels(rng), N=rng.choice([8, 16, 16, 16, 32]),
                    slots=rng.choice([0, B + 7]), dtype=dtype)
    if what == "conv_step":
        B = _log(rng, 1, 128)
        return dict(kind="conv_step", B=B, D=_channels(rng), W=rng.choice([2, 3, 4, 4, 4]),
                    bias=rng.random() < 0.7, silu=rng.random() < 0.8,
                    slots=rng.choice([0, B + 7]), dtype=dtype)
    if what in ("prompt", "packed", "train"):
        D, N = _channels(rng), rng.choice([8, 13, 16, 16, 16, 32])
        most = LARGEST // (D * N) // (1 if what == "train" else 2)
        tokens = _log(rng, 64, min(16384, most))
        lengths = _documents(rng, tokens) if what == "packed" else ""
        B = 1 if what == "packed" else rng.choice([1, 2, 4, 8])
        T = (sum(int(n) for n in lengths.split(",")) if lengths else max(1, tokens // B))
        return dict(kind="scan", B=B, T=T, D=D, N=N, dtype=dtype, train=what == "train",
                    carry=what == "packed" or rng.random() < 0.5, lengths=lengths)
    if what in ("conv", "conv_packed", "conv_train"):
        tokens = _log(rng, 64, 32768)
        lengths = _documents(rng, tokens) if what == "conv_packed" else ""
        B = 1 if what == "conv_packed" else rng.choice([1, 2, 4, 8])
        T = (sum(int(n) for n in lengths.split(",")) if lengths else max(1, tokens // B))
        return dict(kind="conv", B=B, T=T, D=_channels(rng), W=rng.choice([2, 3, 4, 4, 4]),
                    dtype="bf16" if tokens > 16384 else dtype, train=what == "conv_train",
                    carry=rng.random() < 0.5, bias=rng.random() < 0.7, silu=rng.random() < 0.8,
                    lengths=lengths)
    D = rng.choice([64, 64, 80, 96, 128, 128, 256, 70])
    Hk = rng.choice([1, 2, 4, 8, 16])
    Hq = Hk * rng.choice([g for g in (1, 2, 4, 8) if Hk * g <= 32])
    if what == "qk_decode":
        B, T = _log(rng, 1, 128), 1
    else:
        most = 4 * 8192 * 32 * 128 // (D * (Hq + Hk)) // (1 if dtype == "bf16" else 2)
        tokens = _log(rng, 16, min(32768, most))
        B = rng.choice([1, 2, 4])
        T = max(1, tokens // B)
    return dict(kind="qk", B=B, T=T, Hq=Hq, Hk=Hk, D=D, R=rng.choice([D, D, D // 2 // 2 * 2]),
                dtype=dtype, train=what == "qk_train", interleaved=rng.random() < 0.3,
                far=what == "qk_decode" or rng.random() < 0.3)


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


def _ssm_parameters(mk, rand, D, N):
    """Decay rates -1 .. -N and step sizes of 0.001 .. 0.1 as training begins with, a little
    apart from one another as they are later."""
    A = -torch.arange(1, N + 1, device=DEV, dtype=torch.float32) * torch.exp(0.2 * mk(D, N))
    dt = torch.exp(math.log(1e-3) + math.log(100.0) * rand(D))
    return {"A": A, "D": 1.0 + 0.1 * mk(D), "delta_bias": dt + torch.log(-torch.expm1(-dt))}


def _slots(case, gen):
    """(slots of the pool, the batch's slots or None)."""
    if not case["slots"]:
        return case["B"], None
    order = torch.randperm(case["slots"], generator=gen, device=DEV)
    return case["slots"], order[:case["B"]].to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def mk(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=DEV)

    kind, B, D = case["kind"], case["B"], case["D"]
    if kind == "scan_step":
        N = case["N"]
        slots, idx = _slots(case, gen)
        x = {"u": torch.nn.functional.silu(mk(B, D)).to(dt), "delta": (0.5 * mk(B, D)).to(dt),
             "z": mk(B, 2 * D).to(dt)[:, D:]}   # the gate: half of the input projection
        rank = max(1, D // 32)                  # B and C: columns of one projection
        bc = mk(B, rank + 2 * N).to(dt)
        x["B"], x["C"] = bc[:, rank:rank + N], bc[:, rank + N:]
        x.update(_ssm_parameters(mk, rand, D, N))
        return dict(case=case, x=x, idx=idx, state=mk(slots, D, N))
    if kind == "conv_step":
        slots, idx = _slots(case, gen)
        x = {"x": mk(B, 2 * D).to(dt)[:, :D], "weight": (0.5 * mk(D, case["W"])).to(dt),
             "bias": (0.1 * mk(D)).to(dt) if case["bias"] else None}
        return dict(case=case, x=x, idx=idx, state=mk(slots, case["W"], D).to(dt))
    T = case["T"]
    cu = _cu(case)
    S = _sequences(case)
    leaf = (lambda t: t.detach().requires_grad_(case["train"]))   # noqa: E731
    if kind == "scan":
        N = case["N"]
        x = {"u": torch.nn.functional.silu(mk(B, T, D)).to(dt),
             "delta": (0.5 * mk(B, T, D)).to(dt), "z": mk(B, T, 2 * D).to(dt)[..., D:]}
        rank = max(1, D // 32)
        bc = mk(B, T, rank + 2 * N).to(dt)
        x["B"], x["C"] = bc[..., rank:rank + N], bc[..., rank + N:]
        x.update(_ssm_parameters(mk, rand, D, N))
        if case["carry"]:
            x["initial_state"] = mk(S, D, N)
        x = {n: leaf(t) for n, t in x.items()}
        st = dict(case=case, x=x, cu=cu)
        if case["train"]:
            st["dy"] = mk(B, T, D).to(dt)
            st["dht"] = mk(S, D, N) if case["carry"] else None
        return st
    if kind == "conv":
        W = case["W"]
        x = {"x": mk(B, T, 2 * D).to(dt)[..., :D], "weight": (0.5 * mk(D, W)).to(dt)}
        if case["bias"]:
            x["bias"] = (0.1 * mk(D)).to(dt)
        if case["carry"]:
            x["initial_state"] = mk(S, W, D).to(dt)
        x = {n: leaf(t) for n, t in x.items()}
        st = dict(case=case, x=x, cu=cu)
        if case["train"]:
            st["dy"] = mk(B, T, D).to(dt)
            st["dht"] = mk(S, W, D).to(dt) if case["carry"] else None
        return st
    Hq, Hk = case["Hq"], case["Hk"]
    qkv = mk(B, T, Hq + 2 * Hk, D).to(dt)   # the fused projection; v follows the keys
    x = {"q": qkv[:, :, :Hq], "k": qkv[:, :, Hq:Hq + Hk],
         "q_weight": 1.0 + 0.1 * mk(D), "k_weight": 1.0 + 0.1 * mk(D)}
    x = {n: leaf(t) for n, t in x.items()}
    R = case["R"]
    inv_freq = THETA ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R)
    start = torch.randint(0, 1 << 20 if case["far"] else 1, (B, 1), generator=gen, device=DEV)
    st = dict(case=case, x=x, inv_freq=inv_freq,
              positions=start + torch.arange(T, device=DEV)[None])
    if case["train"]:
        st["dq"], st["dk"] = mk(B, T, Hq, D).to(dt), mk(B, T, Hk, D).to(dt)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state)
    with torch.no_grad():
        return {"scan": _scan_plain, "scan_step": _scan_step_plain, "conv": _conv_plain,
                "conv_step": _conv_step_plain, "qk": _qk_plain}[kind](state)


def _own(state):
    """The calls of a user's program."""
    if os.path.join(ROOT, "pallas-kernel_amd") not in sys.path:
        sys.path.insert(0, os.path.join(ROOT, "pallas-kernel_amd"))
    import tops.ops.rope as rope
    import tops.ops.ssm as ssm

    case, x = state["case"], state["x"]
    kind = case["kind"]
    if kind == "scan_step":
        with torch.no_grad():
            y = ssm.selective_scan_step(state["state"], x["u"], x["delta"], x["A"], x["B"], x["C"],
                                        x["D"], z=x["z"], delta_bias=x["delta_bias"],
                                        delta_softplus=True, state_indices=state["idx"])
        return {"y": y, "state": state["state"]}
    if kind == "conv_step":
        with torch.no_grad():
            y = ssm.causal_conv1d_step(x["x"], state["state"], x["weight"], x["bias"],
                                       activation="silu" if case["silu"] else None,
                                       state_indices=state["idx"])
        return {"y": y, "state": state["state"]}
    train = bool(case["train"])
    with torch.set_grad_enabled(train):
        if kind == "qk":
            out = rope.qk_norm_rope(x["q"], x["k"], x["q_weight"], x["k_weight"],
                                    state["inv_freq"], state["positions"], eps=EPS,
                                    interleaved=case["interleaved"])
            names, outs, grads = ["q", "k"], list(out), [state.get("dq"), state.get("dk")]
        else:
            keep = case["carry"]
            if kind == "scan":
                y, ht = ssm.selective_scan(
                    x["u"], x["delta"], x["A"], x["B"], x["C"], x["D"], z=x["z"],
                    delta_bias=x["delta_bias"], delta_softplus=True,
                    initial_state=x.get("initial_state"), output_final_state=keep,
                    cu_seqlens=state["cu"])
            else:
                y, ht = ssm.causal_conv1d(
                    x["x"], x["weight"], x.get("bias"),
                    activation="silu" if case["silu"] else None,
                    initial_state=x.get("initial_state"), output_final_state=keep,
                    cu_seqlens=state["cu"])
            names, outs = ["y", "ht"][:1 + keep], [y, ht][:1 + keep]
            grads = [state.get("dy"), state.get("dht")][:1 + keep]
    res = {n: o.detach() for n, o in zip(names, outs)}
    if train:
        res["grads"] = dict(zip(x, torch.autograd.grad(outs, list(x.values()), grads)))
    return res


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _f(t):
    return None if t is None else t.float()


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _linear_scan(a, b):
    """h_t = a_t h_{t-1} + b_t over dimension 1 from h_{-1} = 0, by doubling: after the pass of
    stride s every row holds the recurrence's last 2s terms."""
    s = 1
    while s < a.shape[1]:
        h, p = b.clone(), a.clone()
        h[:, s:] += a[:, s:] * b[:, :-s]
        p[:, s:] *= a[:, :-s]
        a, b, s = p, h, 2 * s
    return b


def _firsts(state):
    """(rows, tokens) of the first and of the last tokens of the sequences."""
    case, cu = state["case"], state["cu"]
    B, T = case["B"], case["T"]
    if cu is None:
        r = torch.arange(B, device=DEV)
        return r, torch.zeros_like(r), torch.full_like(r, T - 1)
    c = torch.tensor(cu, device=DEV)
    return torch.zeros_like(c[1:]), c[:-1], c[1:] - 1


def _scan_plain(state):
    case = state["case"]
    x = {n: _f(t) for n, t in state["x"].items()}
    dt = DTYPES[case["dtype"]]
    pre = x["delta"] + x["delta_bias"]
    delta = _softplus(pre)
    rows, first, last = _firsts(state)
    a = torch.exp(delta[..., None] * x["A"])
    da = a
    b = (delta * x["u"])[..., None] * x["B"][:, :, None]
    a = a.clone()
    if case["carry"]:
        b[rows, first] += a[rows, first] * x["initial_state"]
    a[rows, first] = 0
    h = _linear_scan(a, b)
    del b
    y = (h * x["C"][:, :, None]).sum(-1) + x["D"] * x["u"]
    sz = _sigmoid(x["z"])
    out = {"y": (y * x["z"] * sz).to(dt)}
    if case["carry"]:
        out["ht"] = h[rows, last].clone()
    if not case["train"]:
        return out
    dout = _f(state["dy"])
    dy = dout * x["z"] * sz
    dz = dout * y * sz * (1 + x["z"] * (1 - sz))
    # g_t = C_t dy_t + a_{t+1} g_{t+1}
    e = x["C"][:, :, None] * dy[..., None]
    if case["carry"]:
        e[rows, last] += _f(state["dht"])
    an = torch.zeros_like(a)
    an[:, :-1] = a[:, 1:]
    g = _linear_scan(an.flip(1), e.flip(1)).flip(1)
    del an, e
    prev = torch.zeros_like(h)
    prev[:, 1:] = h[:, :-1]
    prev[rows, first] = x["initial_state"] if case["carry"] else 0
    gp = g * da * prev
    del prev
    s = (g * x["B"][:, :, None]).sum(-1)
    dpre = (s * x["u"] + (gp * x["A"]).sum(-1)) * _sigmoid(pre)
    grads = {"u": (s * delta + x["D"] * dy).to(dt), "delta": dpre.to(dt), "z": dz.to(dt),
             "B": (g * (delta * x["u"])[..., None]).sum(2).to(dt),
             "C": (h * dy[..., None]).sum(2).to(dt),
             "A": (gp * delta[..., None]).sum((0, 1)), "D": (dy * x["u"]).sum((0, 1)),
             "delta_bias": dpre.sum((0, 1))}
    if case["carry"]:
        grads["initial_state"] = (g * da)[rows, first]
    out["grads"] = {n: grads[n] for n in x}
    return out


def _scan_step_plain(state):
    x = {n: _f(t) for n, t in state["x"].items()}
    idx = slice(None) if state["idx"] is None else state["idx"].long()
    delta = _softplus(x["delta"] + x["delta_bias"])
    h = (state["state"][idx] * torch.exp(delta[..., None] * x["A"])
         + (delta * x["u"])[..., None] * x["B"][:, None])
    state["state"][idx] = h
    y = (h * x["C"][:, None]).sum(-1) + x["D"] * x["u"]
    y = y * x["z"] * _sigmoid(x["z"])
    return {"y": y.to(DTYPES[state["case"]["dtype"]]), "state": state["state"]}


def _windows(state, x, init):
    """The W inputs up to each token, [B, T, D, W]."""
    case, cu = state["case"], state["cu"]
    B, T, D, W = case["B"], case["T"], case["D"], case["W"]
    if cu is None:
        head = x.new_zeros(B, W - 1, D) if init is None else init[:, 1:]
        return torch.cat([head, x], 1).unfold(1, W, 1)
    at, flat = _window_rows(state)
    if init is None:
        init = x.new_zeros(len(cu) - 1, W, D)
    return torch.cat([x[0], init.reshape(-1, D)])[at].reshape(flat).transpose(2, 3)


def _window_rows(state):
    """Packed sequences: the row of each window's inputs in the tokens followed by the states."""
    case = state["case"]
    T, W = case["T"], case["W"]
    c = torch.tensor(state["cu"], device=DEV)
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(c, t, right=True) - 1
    at = t[:, None] + torch.arange(W, device=DEV) - (W - 1)
    before = at - c[seq][:, None]                       # negative: in the state's last rows
    return torch.where(before >= 0, at, T + (seq[:, None] + 1) * W + before), (1, T, W, -1)


def _last_windows(state, x, init):
    """The last W inputs of each sequence, [sequences, W, D]."""
    case, cu = state["case"], state["cu"]
    B, T, W = case["B"], case["T"], case["W"]
    init = torch.zeros(_sequences(case), W, case["D"], device=DEV) if init is None else init
    if cu is None:
        return torch.cat([init, x], 1)[:, -W:]
    return torch.cat([x[0], init.reshape(-1, x.shape[-1])])[_last_rows(state)]


def _last_rows(state):
    case = state["case"]
    T, W = case["T"], case["W"]
    c = torch.tensor(state["cu"], device=DEV)
    at = c[1:, None] - W + torch.arange(W, device=DEV)
    before = at - c[:-1, None]
    seq = torch.arange(len(c) - 1, device=DEV)[:, None]
    return torch.where(before >= 0, at, T + (seq + 1) * W + before)


def _conv_plain(state):
    case = state["case"]
    x = {n: _f(t) for n, t in state["x"].items()}
    dt = DTYPES[case["dtype"]]
    B, T, D, W = case["B"], case["T"], case["D"], case["W"]
    init = x.get("initial_state")
    win = _windows(state, x["x"], init)
    y = (win * x["weight"]).sum(-1)
    if case["bias"]:
        y = y + x["bias"]
    sig = _sigmoid(y)
    out = {"y": (y * sig if case["silu"] else y).to(dt)}
    if case["carry"]:
        out["ht"] = _last_windows(state, x["x"], init).to(dt)
    if not case["train"]:
        return out
    dz = _f(state["dy"])
    if case["silu"]:
        dz = dz * sig * (1 + y * (1 - sig))
    # an input's gradient: the next W tokens' terms, or those before the first one for the state
    ext = torch.nn.functional.pad(dz, (0, 0, W - 1, W - 1)).unfold(1, W, 1)
    dx = (ext * x["weight"].flip(1)).sum(-1)            # inputs -(W - 1) .. T - 1
    dinit, dx = dx[:, :W - 1], dx[:, W - 1:]
    grads = {"weight": (win * dz[..., None]).sum((0, 1)).to(dt)}
    if case["bias"]:
        grads["bias"] = dz.sum((0, 1)).to(dt)
    if case["carry"]:
        full = torch.cat([torch.zeros(B, 1, D, device=DEV), dinit, dx], 1)
        full[:, -W:] += _f(state["dht"])
        grads["initial_state"], dx = full[:, :W].to(dt), full[:, W:]
    grads["x"] = dx.to(dt)
    out["grads"] = {n: grads[n] for n in x}
    return out


def _conv_step_plain(state):
    case = state["case"]
    x = {n: _f(t) for n, t in state["x"].items()}
    idx = slice(None) if state["idx"] is None else state["idx"].long()
    win = torch.cat([state["state"][idx][:, 1:], state["x"]["x"][:, None]], 1)
    state["state"][idx] = win
    y = (win.float() * x["weight"].t()).sum(1)
    if case["bias"]:
        y = y + x["bias"]
    if case["silu"]:
        y = y * _sigmoid(y)
    return {"y": y.to(DTYPES[case["dtype"]]), "state": state["state"]}


def _rotate(t, cos, sin, interleaved):
    """Pairs (i, i + R / 2), or (2 i, 2 i + 1), of the first R columns turned by their angle."""
    R = 2 * cos.shape[-1]
    if interleaved:
        a, b = t[..., 0:R:2], t[..., 1:R:2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = t[..., :R // 2], t[..., R // 2:R]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, t[..., R:]], -1)


def _qk_plain(state):
    case = state["case"]
    x = {n: _f(t) for n, t in state["x"].items()}
    dt = DTYPES[case["dtype"]]
    angle = state["positions"].double()[..., None, None] * state["inv_freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out, grads = {}, {}
    for n in ("q", "k"):
        t, w = x[n], x[n + "_weight"]
        rstd = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
        out[n] = _rotate(t * rstd * w, cos, sin, case["interleaved"]).to(dt)
        if case["train"]:
            d = _rotate(_f(state["d" + n]), cos, -sin, case["interleaved"])
            m = t * rstd
            grads[n + "_weight"] = (d * m).sum((0, 1, 2))
            d = d * w
            grads[n] = (rstd * (d - m * (d * m).mean(-1, keepdim=True))).to(dt)
    if case["train"]:
        out["grads"] = {n: grads[n] for n in x}
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    kind, B, D = case["kind"], case["B"], case["D"]
    if kind == "scan_step":   # u, delta, z in, y out; A, D and the bias; the state in and out
        N = case["N"]
        return {"bytes": 4 * B * D * es + 2 * B * N * es + D * N * 4 + 8 * D + 8 * B * D * N,
                "flops": B * D * (8 * N + 10)}
    if kind == "conv_step":   # W - 1 rows of the window in, W out
        W = case["W"]
        return {"bytes": B * D * es * (2 + 2 * W - 1) + D * es * (W + 1),
                "flops": B * D * (2 * W + 4)}
    tok = B * case["T"]
    S = _sequences(case) if kind != "qk" else 0
    if kind == "scan":
        N = case["N"]
        states = 4 * S * D * N if case["carry"] else 0
        small = 4 * D * N + 8 * D
        if not case["train"]:
            return {"bytes": 4 * tok * D * es + 2 * tok * N * es + small + 2 * states,
                    "flops": tok * D * (8 * N + 10)}
        return {"bytes": 8 * tok * D * es + 4 * tok * N * es + 2 * small + 4 * states,
                "flops": tok * D * (22 * N + 30)}
    if kind == "conv":
        W = case["W"]
        states = S * W * D * es if case["carry"] else 0
        small = D * (W + case["bias"]) * es
        if not case["train"]:
            return {"bytes": 2 * tok * D * es + small + 2 * states,
                    "flops": tok * D * (2 * W + 4)}
        return {"bytes": 4 * tok * D * es + 2 * small + 4 * states,
                "flops": tok * D * (8 * W + 14)}
    n = tok * (case["Hq"] + case["Hk"]) * D
    small = 8 * D + 8 * tok + 4 * case["R"]
    if not case["train"]:
        return {"bytes": 2 * n * es + small, "flops": 7 * n}
    return {"bytes": 4 * n * es + small + 8 * D, "flops": 20 * n}


# ---------------------------------------------------------------------------
# the same values in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    x = {n: None if t is None else t.detach().double() for n, t in st["x"].items()}
    kind = case["kind"]
    if kind == "scan":
        return _scan64(case, st, x)
    if kind == "scan_step":
        return _scan_step64(st, x)
    if kind == "conv_step":
        return _conv_step64(case, st, x)
    train = bool(case["train"])
    leaves = {n: t.requires_grad_(train) for n, t in x.items()}
    with torch.set_grad_enabled(train):
        outs = _conv64(case, st, leaves) if kind == "conv" else _qk64(case, st, leaves)
    res = {n: o.detach() for n, o in outs.items()}
    if train:
        ups = {"y": "dy", "ht": "dht", "q": "dq", "k": "dk"}
        up = [st[ups[n]].double() for n in outs]
        grads = torch.autograd.grad(list(outs.values()), list(leaves.values()), up)
        res["grads"] = dict(zip(leaves, grads))
    return res


def _scan64(case, st, x):
    """The recurrence token by token, and its adjoint in the reverse order."""
    B, T, D, N = (case[n] for n in "BTDN")
    cu = st["cu"]
    starts = {0} if cu is None else set(cu[:-1])
    ends = {T - 1} if cu is None else {c - 1 for c in cu[1:]}
    pre = x["delta"] + x["delta_bias"]
    delta = torch.nn.functional.softplus(pre, threshold=1e9)
    init = x.get("initial_state")
    silu = torch.nn.functional.silu
    h = torch.zeros(B, D, N, dtype=torch.float64, device=DEV)
    hs, y, ht, seq = [], torch.empty_like(delta), [], 0
    for t in range(T):
        if t in starts:
            h = torch.zeros_like(h) if init is None else init if cu is None else init[seq:seq + 1]
            seq += 1
        if case["train"]:
            hs.append(h)
        d = delta[:, t, :, None]
        h = torch.exp(d * x["A"]) * h + d * x["B"][:, t, None] * x["u"][:, t, :, None]
        y[:, t] = (h * x["C"][:, t, None]).sum(-1)
        if t in ends:
            ht.append(h)
    y = y + x["D"] * x["u"]
    out = {"y": y * silu(x["z"])}
    if case["carry"]:
        out["ht"] = torch.cat(ht)
    if not case["train"]:
        return out
    dout = st["dy"].double()
    sz = torch.sigmoid(x["z"])
    dy = dout * silu(x["z"])
    grads = {n: torch.zeros_like(t) for n, t in x.items()}
    grads["z"] = dout * y * (sz + x["z"] * sz * (1 - sz))
    grads["u"] = dy * x["D"]
    grads["D"] = (dy * x["u"]).sum((0, 1))
    c = torch.zeros(B, D, N, dtype=torch.float64, device=DEV)
    if case["carry"]:
        c = c + st["dht"].double()
    ddelta = torch.empty_like(delta)
    for t in reversed(range(T)):
        d, u, prev = delta[:, t, :, None], x["u"][:, t, :, None], hs.pop()
        bt, ct = x["B"][:, t, None], x["C"][:, t, None]
        a = torch.exp(d * x["A"])
        h = a * prev + d * bt * u
        grads["C"][:, t] = (h * dy[:, t, :, None]).sum(1)
        c = c + ct * dy[:, t, :, None]
        grads["B"][:, t] = (c * d * u).sum(1)
        grads["u"][:, t] += (c * bt * d).sum(-1)
        ga = c * prev * a
        ddelta[:, t] = (ga * x["A"] + c * bt * u).sum(-1)
        grads["A"] += (ga * d).sum(0)
        c = c * a
    grads["delta"] = ddelta * torch.sigmoid(pre)
    grads["delta_bias"] = grads["delta"].sum((0, 1))
    if case["carry"]:
        grads["initial_state"] = c
    out["grads"] = grads
    return out


def _scan_step64(st, x):
    state = st["state"].double()
    idx = torch.arange(len(x["u"]), device=DEV) if st["idx"] is None else st["idx"].long()
    d = torch.nn.functional.softplus(x["delta"] + x["delta_bias"], threshold=1e9)
    h = torch.exp(torch.einsum("bd,dn->bdn", d, x["A"])) * state[idx]
    h = h + torch.einsum("bd,bd,bn->bdn", d, x["u"], x["B"])
    state[idx] = h
    y = torch.einsum("bdn,bn->bd", h, x["C"]) + x["D"] * x["u"]
    return {"y": y * torch.nn.functional.silu(x["z"]), "state": state}


def _conv64(case, st, x):
    """Sequence by sequence, tap by tap."""
    W, cu = case["W"], st["cu"]
    init = x.get("initial_state")
    rows = x["x"].unbind(0) if cu is None else [x["x"][0, a:b] for a, b in zip(cu, cu[1:])]
    ys, ends = [], []
    for i, row in enumerate(rows):
        head = row.new_zeros(W, row.shape[1]) if init is None else init[i]
        row = torch.cat([head, row])
        n = len(row) - W
        z = sum(row[1 + j:1 + j + n] * x["weight"][:, j] for j in range(W))
        if case["bias"]:
            z = z + x["bias"]
        ys.append(torch.nn.functional.silu(z) if case["silu"] else z)
        ends.append(row[n:])
    out = {"y": torch.stack(ys) if cu is None else torch.cat(ys)[None]}
    if case["carry"]:
        out["ht"] = torch.stack(ends)
    return out


def _conv_step64(case, st, x):
    state = st["state"].double()
    idx = torch.arange(len(x["x"]), device=DEV) if st["idx"] is None else st["idx"].long()
    state[idx] = torch.cat([state[idx, 1:], x["x"][:, None]], 1)
    y = torch.einsum("bwd,dw->bd", state[idx], x["weight"])
    if case["bias"]:
        y = y + x["bias"]
    return {"y": torch.nn.functional.silu(y) if case["silu"] else y, "state": state}


def _qk64(case, st, x):
    """The rotation as a product of complex numbers."""
    R = case["R"]
    ph = torch.polar(torch.ones_like(st["inv_freq"]).expand(*st["positions"].shape, -1),
                     st["positions"].double()[..., None] * st["inv_freq"])[:, :, None]
    out = {}
    for n in ("q", "k"):
        t = x[n] / torch.sqrt(x[n].square().mean(-1, keepdim=True) + EPS) * x[n + "_weight"]
        pairs = t[..., :R].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
        dim = -1 if case["interleaved"] else -2
        c = torch.complex(*pairs.unbind(dim)) * ph
        out[n] = torch.cat([torch.stack([c.real, c.imag], dim).flatten(-2), t[..., R:]], -1)
    return out
