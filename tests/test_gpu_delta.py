"""gated_delta_rule and gated_delta_rule_step against the recurrence in 64 bits (bounds: delta_ref)."""

import pytest
import torch
import torch.nn.functional as F

from delta_ref import F64, HALF, ULP32, bound, close, delta
from tops.ops.delta import gated_delta_rule, gated_delta_rule_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FL = torch.bfloat16, torch.float32
NAMES = ("q", "k", "v", "g", "beta", "initial_state")


def make(B, T, H, HV, K, V, dt, S=None, init=True, norm=False, seed=0, gdt=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)   # noqa: E731
    gdt = dt if gdt is None else gdt
    size = 1.0 if norm else K ** -0.5
    x = dict(q=r(B, T, H, K).to(dt), k=(size * r(B, T, H, K)).to(dt), v=r(B, T, HV, V).to(dt),
             g=(-0.3 * r(B, T, HV).abs()).to(gdt), beta=torch.sigmoid(r(B, T, HV)).to(gdt),
             initial_state=r(B if S is None else S, HV, K, V) if init else None)
    return x, r


def check(x, r, cu=None, norm=False, scale=None, to=lambda n, t: t.to(DEV), want=NAMES, dht=True,
          tol=1.0):
    dt = x["q"].dtype
    B, T, H, K = x["q"].shape
    names = [n for n in NAMES if x[n] is not None]
    d = {n: to(n, x[n]).detach().requires_grad_(n in want) for n in names}
    o, ht = gated_delta_rule(**d, scale=scale, output_final_state=True, cu_seqlens=cu,
                             qk_l2norm=norm)
    assert o.dtype == dt and ht.dtype == FL
    do, dh = r(*o.shape).to(dt), r(*ht.shape)
    c = {n: x[n].to(F64).requires_grad_() for n in names}
    ro, rht = delta(c["q"], c["k"], c["v"], c["g"], c["beta"], c.get("initial_state"), scale, cu,
                    norm)
    tokens = T if cu is None else max([1, *(b - a for a, b in zip(cu, cu[1:]))])
    b = lambda n: tol * bound(n, dt, K, tokens)   # noqa: E731
    close("o", o, ro, b("o"))
    close("ht", ht, rht, b("ht"))
    asked = [n for n in names if n in want]
    outs, ups, refs = [o, ht][:1 + dht], [do.to(DEV), dh.to(DEV)][:1 + dht], [ro, rht][:1 + dht]
    got = torch.autograd.grad(outs, [d[n] for n in asked], ups)
    some = [(t, u.cpu().to(F64)) for t, u in zip(refs, ups) if t.requires_grad]   # of any token
    ref = ([None] * len(asked) if not some else
           torch.autograd.grad([t for t, _ in some], [c[n] for n in asked],
                               [u for _, u in some], allow_unused=True))
    for n, t, w in zip(asked, got, ref):
        assert t.dtype == d[n].dtype and t.shape == d[n].shape, n
        w = torch.zeros_like(c[n]) if w is None else w
        # dg is a difference of sums of the terms o . do, ht . dht and n . dn (n <= v, dn near dv),
        # whose float32 roundings stay where they cancel: before a sequence's first token there is
        # no state that a decay could matter to, and dg is exactly 0
        floor = 1e-30
        if n == "g" and "v" in asked:
            dv = got[asked.index("v")]
            pairs = ((ro, do), (rht, dh), (x["v"], dv), (x["v"], dv))
            floor = bound("o", FL, K, tokens) * sum(
                a.detach().double().norm().item() * c.double().norm().item() for a, c in pairs)
        # a gradient returned in another type than its terms are computed in
        close("d" + n, t, w, b(n) + (HALF if t.dtype is BF and dt is FL else 0), floor)
    return o, ht, got


# tokens around a chunk (64, in float32 32) and its halves, head sizes around the padded ones
@pytest.mark.parametrize("B,T,H,HV,K,V", [
    (1, 1, 1, 1, 64, 32), (2, 31, 1, 2, 64, 64), (1, 33, 2, 2, 128, 16), (2, 64, 1, 1, 32, 128),
    (1, 65, 2, 4, 64, 72), (1, 130, 1, 3, 128, 40), (1, 200, 1, 1, 256, 64), (1, 97, 1, 2, 200, 24)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dt", [FL, BF])
def test_forward_backward(B, T, H, HV, K, V, norm, dt):
    x, r = make(B, T, H, HV, K, V, dt, norm=norm)
    check(x, r, norm=norm)


# sizes that no piece of 8 divides, fewer than 8 of them, and many columns
@pytest.mark.parametrize("K,V", [(1, 1), (3, 20), (20, 5), (9, 9), (65, 33), (99, 130), (129, 17),
                                 (255, 15), (16, 300)])
@pytest.mark.parametrize("dt", [FL, BF])
def test_odd_sizes(K, V, dt):
    x, r = make(2, 70, 1, 2, K, V, dt, norm=K > 2)
    check(x, r, norm=K > 2)


@pytest.mark.parametrize("lens", [[1], [2, 1, 64, 30], [0, 7, 0, 0, 65, 0], [0, 0],
                                  [3, 128, 3, 100, 64]])
@pytest.mark.parametrize("init", [True, False])
@pytest.mark.parametrize("dt", [FL, BF])
def test_packed(lens, init, dt):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x, r = make(1, cu[-1], 1, 2, 64, 40, dt, S=len(lens), init=init, norm=True)
    check(x, r, cu=cu, norm=True)


@pytest.mark.parametrize("lens", [[1100], [1500, 20, 700, 0, 300, 64], [1025]])
@pytest.mark.parametrize("K,V", [(64, 20), (100, 90)])
@pytest.mark.parametrize("dt", [FL, BF])
def test_segments(lens, K, V, dt):
    """Sequences long enough to be cut into segments that run in parallel."""
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x, r = make(1, cu[-1], 1, 2, K, V, dt, S=len(lens), norm=True)
    x["g"] *= 0.05   # what is before a segment has to matter at its end
    check(x, r, cu=cu, norm=True)
    if len(lens) == 1:
        check(x, r, norm=True)


@pytest.mark.parametrize("lens", [[400], [130] * 10 + [900, 0, 640]])
@pytest.mark.parametrize("dt", [FL, BF])
def test_segments_of_few_chunks_and_of_many_sequences(lens, dt):
    """Two chunks a segment; and more blocks than run at once, long sequences among short ones."""
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x, r = make(1, cu[-1], 3, 6, 32, 500, dt, S=len(lens), norm=True)
    x["g"] *= 0.05
    check(x, r, cu=cu, norm=True)


@pytest.mark.parametrize("value", [-50.0, float(torch.finfo(FL).min), -torch.inf])
@pytest.mark.parametrize("dt", [FL, BF])
def test_strong_decays_over_segments(value, dt):
    """A segment that forgets all before it, at its first, last or another token, and one that
    does not."""
    x, r = make(1, 1000, 1, 2, 64, 32, dt, norm=True, gdt=FL)
    x["g"] *= 0.05
    x["g"][:, [128, 255, 300, 511, 512, 513]] = value
    if value == -torch.inf:   # the oracle's gradients of these decays are inf * 0
        d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
        o, ht = gated_delta_rule(**d, output_final_state=True, qk_l2norm=True)
        grads = torch.autograd.grad([o, ht], list(d.values()),
                                    [torch.ones_like(o), torch.ones_like(ht)])
        assert all(torch.isfinite(t).all() for t in grads)
        x["g"].clamp_(min=-1000.0)   # e^-1000 is 0 in the oracle too
    check(x, r, norm=True)


def test_packed_sequences_are_independent():
    """Inputs of a sequence that are not finite leave the others' outputs, final states and
    gradients as they are, with segments and without."""
    lens = [70, 900, 60, 800, 3]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x, r = make(1, cu[-1], 1, 2, 64, 32, BF, S=len(lens), norm=True)
    up = r(1, cu[-1], 2, 32).to(BF).to(DEV), r(len(lens), 2, 64, 32).to(DEV)

    def run(**bad):
        d = {n: t.to(DEV) for n, t in x.items()}
        for n, (i, b) in bad.items():
            d[n][0, i] = b
        d = {n: t.requires_grad_() for n, t in d.items()}
        o, ht = gated_delta_rule(**d, output_final_state=True, cu_seqlens=cu, qk_l2norm=True)
        *grads, dh = torch.autograd.grad([o, ht], list(d.values()), up)
        tokens = [t.split(lens, 1) for t in (o, *grads)]
        return [[ht[s], dh[s], *(t[s] for t in tokens)] for s in range(len(lens))]

    want = run()
    for name, bad in (("v", torch.inf), ("k", torch.nan), ("g", torch.inf), ("beta", torch.nan)):
        for s in (1, 2):   # a sequence of segments, and one without
            got = run(**{name: (cu[s] + 30, bad)})
            assert not torch.isfinite(got[s][0]).all()
            for e in range(len(lens)):
                if e != s:
                    assert all(torch.equal(a, b) for a, b in zip(want[e], got[e])), (name, s, e)


@pytest.mark.parametrize("B,T", [(0, 5), (2, 0), (0, 0)])
@pytest.mark.parametrize("dt", [FL, BF])
def test_no_tokens(B, T, dt):
    x, r = make(B, T, 1, 2, 64, 16, dt)
    o, ht, got = check(x, r)
    assert torch.equal(ht.cpu(), x["initial_state"])


@pytest.mark.parametrize("want", [("q",), ("v", "beta"), ("initial_state",), ("g", "k")])
@pytest.mark.parametrize("dht", [True, False])
def test_some_gradients(want, dht):
    x, r = make(1, 80, 1, 2, 64, 32, FL)
    check(x, r, want=want, dht=dht)


def test_only_the_final_state_has_a_gradient():
    x, r = make(1, 80, 1, 2, 64, 32, BF)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    _, ht = gated_delta_rule(**d, output_final_state=True)
    dh = r(*ht.shape)
    c = {n: t.to(F64).requires_grad_() for n, t in x.items()}
    ref = delta(c["q"], c["k"], c["v"], c["g"], c["beta"], c["initial_state"])[1]
    names = [n for n in NAMES if n != "q"]
    got = torch.autograd.grad(ht, [d[n] for n in NAMES], dh.to(DEV))
    want = torch.autograd.grad(ref, [c[n] for n in names], dh.to(F64))
    assert not got[0].any()
    for n, t, w in zip(names, got[1:], want):
        close("d" + n, t, w, bound(n, BF, 64, 80))


@pytest.mark.parametrize("value", [0.0, -50.0, -1000.0, float(torch.finfo(FL).min), -torch.inf])
@pytest.mark.parametrize("dt", [FL, BF])
def test_strong_decays(value, dt):
    """Some tokens forget nearly all, or all. The oracle's float64 has e^-inf = 0 too."""
    x, r = make(1, 150, 1, 2, 64, 32, dt, norm=True, gdt=FL)
    x["g"][:, ::7] = value
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    o, ht = gated_delta_rule(**d, output_final_state=True, qk_l2norm=True)
    c = {n: t.to(F64).requires_grad_() for n, t in x.items()}
    ro, rht = delta(c["q"], c["k"], c["v"], c["g"], c["beta"], c["initial_state"], l2norm=True)
    close("o", o, ro, bound("o", dt, 64, 150))
    close("ht", ht, rht, bound("ht", dt, 64, 150))
    do, dh = r(*o.shape).to(dt), r(*ht.shape)
    got = torch.autograd.grad([o, ht], list(d.values()), [do.to(DEV), dh.to(DEV)])
    ref = torch.autograd.grad([ro, rht], list(c.values()), [do.to(F64), dh.to(F64)])
    for n, t, w in zip(d, got, ref):
        w = torch.nan_to_num(w) if value == -torch.inf else w
        close("d" + n, t, w, bound(n, dt, 64, 150))


@pytest.mark.parametrize("value", [0.0, 1e-30, 2.0, -0.5])
@pytest.mark.parametrize("dt", [FL, BF])
def test_written_strengths(value, dt):
    """Tokens that write nothing still have a gradient of beta."""
    x, r = make(1, 100, 1, 2, 64, 32, dt, norm=True, gdt=FL)
    x["beta"][:, ::3] = value
    check(x, r, norm=True)


@pytest.mark.parametrize("dt", [FL, BF])
def test_equal_keys(dt):
    """One key for all tokens, beta = 1: every token replaces what the one before wrote, and the
    triangular system is as far from the identity as it can be."""
    x, r = make(1, 130, 1, 1, 64, 32, dt, gdt=FL)
    x["k"] = F.normalize(x["k"][:, :1].float(), dim=-1).to(dt).expand(1, 130, 1, 64).clone()
    x["beta"] = torch.ones(1, 130, 1)
    x["g"] = torch.zeros(1, 130, 1)
    check(x, r, norm=True)


@pytest.mark.parametrize("gdt,bdt", [(FL, BF), (BF, FL), (torch.float16, F64)])
def test_types_of_gates(gdt, bdt):
    x, r = make(1, 70, 1, 2, 64, 32, BF)
    x["g"], x["beta"] = x["g"].to(gdt), x["beta"].to(bdt)
    check(x, r)


def test_half_inputs():
    """float16 is computed in float32 and rounded at the end."""
    x, r = make(1, 70, 1, 2, 64, 32, torch.float16)
    d = {n: t.to(DEV) for n, t in x.items()}
    o, _ = gated_delta_rule(**d)
    ro, _ = delta(*(x[n].to(F64) for n in NAMES))
    assert o.dtype == torch.float16
    close("o", o, ro, 2.0 ** -11 + bound("o", FL, 64, 70))


@pytest.mark.parametrize("dt", [FL, BF])
def test_views(dt):
    """Queries, keys and values side by side in one row, gates as columns of another."""
    x, r = make(2, 70, 2, 4, 24, 40, dt)

    def view(n, t):
        t = t.to(DEV)
        if n in "qkv":
            wide = torch.zeros(*t.shape[:2], 3 * t.shape[2] * t.shape[3] + 1, dtype=t.dtype,
                               device=DEV)
            at = wide[..., 1 + t.shape[2] * t.shape[3]:1 + 2 * t.shape[2] * t.shape[3]]
            at.copy_(t.flatten(2))
            return at.unflatten(-1, t.shape[2:])
        if n in ("g", "beta"):
            return torch.cat([t, t], -1)[..., t.shape[-1]:]
        return t

    check(x, r, to=view)
    check(x, r, to=lambda n, t: t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
          if n in NAMES[:5] else t.to(DEV))
    check(x, r, to=lambda n, t: t.to(DEV).transpose(-1, -2).contiguous().transpose(-1, -2))


def test_upstream_views():
    """The gradient of o as an expanded tensor and as a transposed one."""
    x, r = make(1, 70, 1, 2, 64, 32, BF)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    o, _ = gated_delta_rule(**d)
    one = torch.autograd.grad(o.float().sum(), list(d.values()), retain_graph=True)
    two = torch.autograd.grad(o, list(d.values()),
                              torch.ones(1, 2, 70, 32, dtype=BF, device=DEV).transpose(1, 2))
    assert all(torch.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize("dt", [FL, BF])
def test_pieces_and_steps_go_on(dt):
    """A prompt in three pieces, then tokens one by one and four at once, as the whole."""
    x, _ = make(2, 150, 1, 2, 64, 32, dt, norm=True, gdt=FL)
    d = {n: t.to(DEV) for n, t in x.items()}
    ro, rht = delta(*(x[n].to(F64) for n in NAMES), l2norm=True)
    h, outs = d["initial_state"], []
    cut = lambda a, b: [d[n][:, a:b] for n in NAMES[:5]]   # noqa: E731
    for a, b in ((0, 1), (1, 90), (90, 140)):
        o, h = gated_delta_rule(*cut(a, b), initial_state=h, output_final_state=True,
                                qk_l2norm=True)
        outs.append(o)
    with torch.no_grad():
        for t in range(140, 146):
            o = gated_delta_rule_step(h, *(y[:, 0] for y in cut(t, t + 1)), qk_l2norm=True)
            outs.append(o[:, None])
        outs.append(gated_delta_rule_step(h, *cut(146, 150), qk_l2norm=True))
    close("o", torch.cat(outs, 1), ro, bound("o", dt, 64, 150))
    close("ht", h, rht, 3 * bound("ht", dt, 64, 150))


def test_repeats_are_equal():
    x, r = make(2, 300, 2, 4, 128, 64, BF, norm=True)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    do = r(2, 300, 4, 64).to(BF).to(DEV)
    runs = []
    for _ in range(3):
        o, ht = gated_delta_rule(**d, output_final_state=True, qk_l2norm=True)
        runs.append([o, ht, *torch.autograd.grad([o, ht], list(d.values()),
                                                 [do, torch.ones_like(ht)])])
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))


def test_rows_are_independent():
    """A batch row with inputs that are not finite leaves the others as they are."""
    x, _ = make(3, 70, 1, 2, 64, 32, BF)
    d = {n: t.to(DEV) for n, t in x.items()}
    o, ht = gated_delta_rule(**d, output_final_state=True)
    for n, bad in (("v", torch.inf), ("k", torch.nan), ("g", torch.inf)):
        e = {m: t.clone() for m, t in d.items()}
        e[n][1, 5] = bad
        o2, ht2 = gated_delta_rule(**e, output_final_state=True)
        assert torch.equal(o[::2], o2[::2]) and torch.equal(ht[::2], ht2[::2])
        assert not torch.isfinite(o2[1]).all()


# ---------------------------------------------------------------------------
# streams, graphs, size
# ---------------------------------------------------------------------------


def test_streams():
    x, r = make(1, 400, 2, 2, 128, 128, BF, norm=True)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    do = r(1, 400, 2, 128).to(BF).to(DEV)

    def call():
        o, _ = gated_delta_rule(**d, qk_l2norm=True)
        return [o, *torch.autograd.grad(o, list(d.values()), do)]

    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(want, g))


@pytest.mark.parametrize("cu", [None, [0, 10, 10, 250]])
def test_captured(cu):
    """Forward and backward in a graph, replayed with eager work between."""
    x, r = make(1, 250, 1, 2, 64, 64, BF, S=1 if cu is None else 3, norm=True)
    d = {n: t.to(DEV).requires_grad_() for n, t in x.items()}
    do = r(1, 250, 2, 64).to(BF).to(DEV)

    def call():
        o, ht = gated_delta_rule(**d, output_final_state=True, cu_seqlens=cu, qk_l2norm=True)
        return [o.detach(), ht.detach(), *torch.autograd.grad([o, ht], list(d.values()),
                                                              [do, torch.ones_like(ht)])]

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        with torch.no_grad():
            for n in ("q", "v"):
                d[n].mul_(0.7).add_(0.1 * i)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), i


def test_two_graphs_and_eager_calls_in_turn():
    """Two captured calls, one of segments, replayed in turn with eager calls between."""
    runs = []
    for T, K in ((70, 64), (700, 128)):
        x, _ = make(1, T, 1, 2, K, 64, BF, norm=True)
        d = {n: t.to(DEV) for n, t in x.items()}
        call = lambda d=d: gated_delta_rule(   # noqa: E731
            **d, output_final_state=True, qk_l2norm=True)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        runs.append((d, call, graph, out))
    for i in range(4):
        for d, *_ in runs:
            d["v"].mul_(0.7).add_(0.1 * i)
        for _, _, graph, _ in runs:
            graph.replay()
        for _, call, _, out in runs:
            assert all(torch.equal(a, b) for a, b in zip(call(), out)), i


def test_packed_lengths_new_to_a_capture_raise():
    x, _ = make(1, 61, 1, 1, 64, 16, BF, S=2)
    d = {n: t.to(DEV) for n, t in x.items()}
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gated_delta_rule(**d, cu_seqlens=[0, 17, 61])
    torch.cuda.synchronize()


def test_rows_past_2_31_elements():
    """A sequence whose queries, keys and values lie past 2^31 elements, as alone."""
    T, H, K = (1 << 31) // (16 * 128) + 500, 16, 128
    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV, dtype=BF)   # noqa: E731
    q, k, v = (r(1, T, H, K) for _ in range(3))
    g, beta = -0.1 * r(1, T, H).abs(), torch.sigmoid(r(1, T, H))
    cu = [0, 1 << 19, T - 130, T]
    with torch.no_grad():
        o, ht = gated_delta_rule(q, k, v, g, beta, output_final_state=True, cu_seqlens=cu,
                                 qk_l2norm=True)
        alone, hta = gated_delta_rule(*(t[:, -130:] for t in (q, k, v, g, beta)),
                                      output_final_state=True, qk_l2norm=True)
    assert torch.equal(o[:, -130:], alone) and torch.equal(ht[2:], hta)


# ---------------------------------------------------------------------------
# the step
# ---------------------------------------------------------------------------


def step_check(x, slots=None, idx=None, norm=False, to=lambda n, t: t.to(DEV), scale=None):
    """x with T tokens; the step's bound: float32 sums over the keys, one more rounding a token."""
    dt = x["q"].dtype
    B, T, H, K = x["q"].shape
    slots = B if slots is None else slots
    gen = torch.Generator().manual_seed(9)
    pool = torch.randn(slots, *x["initial_state"].shape[1:], generator=gen)
    where = list(range(B)) if idx is None else idx
    rows = [(b, s) for b, s in enumerate(where) if 0 <= s < slots]
    want_o = torch.zeros(*x["v"].shape, dtype=F64)
    want_h = pool.to(F64)
    if rows:
        take = lambda n: x[n][[b for b, _ in rows]].to(F64)   # noqa: E731
        at = [s for _, s in rows]
        o, h = delta(*(take(n) for n in NAMES[:5]), pool[at].to(F64), scale, None, norm)
        want_o[[b for b, _ in rows]] = o
        want_h[at] = h
    tol = (K + 16 + 4 * T) * ULP32 * 2
    for one in ((True, False) if T == 1 else (False,)):
        state = pool.to(DEV)
        v0 = state._version
        args = [to(n, x[n]) for n in NAMES[:5]]
        args = [t[:, 0] for t in args] if one else args
        t = None if idx is None else torch.tensor(idx, dtype=torch.int32, device=DEV)
        with torch.no_grad():
            got = gated_delta_rule_step(state, *args, scale=scale, qk_l2norm=norm, state_indices=t)
        assert got.dtype == dt and got.shape == args[2].shape
        assert state._version == v0 + 1
        got = got[:, None] if one else got
        close("o", got, want_o, tol + (HALF if dt is BF else 0))
        close("state", state, want_h, tol)
        for s in set(range(slots)) - {s for _, s in rows}:
            assert torch.equal(state[s].cpu(), pool[s])
        for b in set(range(B)) - {b for b, _ in rows}:
            assert not got[b].any()


@pytest.mark.parametrize("B,T,H,HV,K,V", [
    (1, 1, 1, 1, 64, 16), (3, 1, 2, 4, 128, 128), (2, 4, 1, 3, 128, 72), (2, 3, 1, 1, 256, 64),
    (1, 1, 1, 2, 1, 1), (2, 2, 1, 1, 7, 3), (2, 1, 1, 2, 99, 33), (1, 2, 1, 1, 200, 130),
    (2, 9, 1, 1, 65, 20)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dt", [FL, BF])
def test_step(B, T, H, HV, K, V, norm, dt):
    x, _ = make(B, T, H, HV, K, V, dt, norm=norm)
    step_check(x, norm=norm)


@pytest.mark.parametrize("idx", [[4, 0, 2], [5, -1, 1], [-1, -7, 9], [6, 3, 2 ** 31 - 1]])
def test_step_slots(idx):
    x, _ = make(3, 2, 1, 2, 64, 40, BF)
    step_check(x, slots=6, idx=idx)


def test_step_wide_indices_and_strided_pool():
    x, _ = make(2, 1, 1, 2, 64, 32, BF)
    d = {n: t.to(DEV)[:, 0] for n, t in x.items() if n != "initial_state"}
    wide = torch.randn(5, 3, 2, 64, 32, device=DEV)
    state, other = wide[:, 1], wide.clone()
    ref = state.clone()
    idx = torch.tensor([3, 1], device=DEV)
    with torch.no_grad():
        a = gated_delta_rule_step(state, **d, state_indices=idx)
        b = gated_delta_rule_step(ref, **d, state_indices=idx.int())
    assert torch.equal(a, b) and torch.equal(state, ref)
    assert torch.equal(wide[:, ::2], other[:, ::2])


def test_step_views_and_scale():
    x, _ = make(2, 3, 2, 4, 24, 40, BF, gdt=FL)
    pad = lambda n, t: torch.cat([t, t], -1).to(DEV)[..., t.shape[-1]:]   # noqa: E731
    step_check(x, to=pad, scale=0.3)
    step_check(x, to=lambda n, t: t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1),
               norm=True)
    step_check(x, to=lambda n, t: t.to(DEV).transpose(-1, -2).contiguous().transpose(-1, -2))


def test_step_no_rows():
    x, _ = make(0, 1, 1, 2, 64, 32, BF)
    d = {n: t.to(DEV)[:, 0] for n, t in x.items() if n != "initial_state"}
    with torch.no_grad():
        state = torch.randn(3, 2, 64, 32, device=DEV)
        before = state.clone()
        assert gated_delta_rule_step(state, **d).shape == (0, 2, 32)
        x, _ = make(3, 0, 1, 2, 64, 32, BF)
        d = {n: t.to(DEV) for n, t in x.items() if n != "initial_state"}
        assert gated_delta_rule_step(state, **d).shape == (3, 0, 2, 32)
    assert torch.equal(state, before)


def test_step_forgets():
    x, _ = make(2, 1, 1, 2, 64, 32, FL)
    x["g"][0] = -torch.inf
    step_check(x)


def test_step_captured():
    x, _ = make(3, 1, 1, 2, 64, 32, BF, norm=True)
    d = {n: t.to(DEV)[:, 0] for n, t in x.items() if n != "initial_state"}
    state, eager = (torch.ones(5, 2, 64, 32, device=DEV) for _ in range(2))
    idx = torch.tensor([4, 0, 2], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        call = lambda s: gated_delta_rule_step(s, **d, qk_l2norm=True, state_indices=idx)  # noqa: E731
        call(state.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(state)
        for i in range(4):
            idx.copy_((idx + 1) % 5)
            d["v"].add_(0.25)
            want = call(eager)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(state, eager), i


def test_step_slots_past_2_31_elements():
    slots = (1 << 31) // (8 * 128 * 128) + 2
    state = torch.zeros(slots, 8, 128, 128, device=DEV)
    x, _ = make(1, 1, 8, 8, 128, 128, BF)
    d = {n: t.to(DEV)[:, 0] for n, t in x.items() if n != "initial_state"}
    ref = torch.zeros(1, 8, 128, 128, device=DEV)
    with torch.no_grad():
        idx = torch.tensor([slots - 1], device=DEV)
        a = gated_delta_rule_step(state, **d, state_indices=idx)
        b = gated_delta_rule_step(ref, **d)
    assert torch.equal(a, b) and torch.equal(state[-1:], ref)
