"""How far an input that is not finite reaches: what gated_delta_rule's documentation says of it."""

import pytest
import torch

from tops.ops.delta import gated_delta_rule

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FL = torch.bfloat16, torch.float32
B, T, H, HV, K, V = 2, 200, 2, 4, 64, 40
ROW, AT, HEAD, COL = 1, 70, 1, 5   # batch row, token, key head (or its first value head), column


def inputs(dt):
    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)   # noqa: E731
    x = dict(q=r(B, T, H, K).to(dt), k=r(B, T, H, K).to(dt), v=r(B, T, HV, V).to(dt),
             g=-0.1 * r(B, T, HV).abs(), beta=torch.sigmoid(r(B, T, HV)),
             initial_state=r(B, HV, K, V))
    return x, r(B, T, HV, V).to(dt), r(B, HV, K, V)


def reach(name):
    """Of o and the final state, what is not finite: of the value heads of a key head the token and all
    that follow, and less for q and v."""
    o, ht = (torch.zeros(B, n, HV, V, dtype=torch.bool, device=DEV) for n in (T, K))
    ht = ht.transpose(1, 2).contiguous()
    heads = slice(2 * HEAD, 2 * HEAD + 2) if name in "qk" else slice(2 * HEAD, 2 * HEAD + 1)
    cols = slice(COL, COL + 1) if name == "v" else slice(None)
    if name == "q":
        o[ROW, AT, heads] = True
    else:
        o[ROW, AT:, heads, cols] = True
        ht[ROW, heads, :, cols] = True
    return o, ht


def spoil(x, name, bad):
    x = {n: t.clone() for n, t in x.items()}
    at = HEAD if name in "qk" else 2 * HEAD
    t = x[name]
    t[(ROW, AT, at, COL)[:t.dim()]] = bad
    return x


@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta"])
@pytest.mark.parametrize("bad", [torch.inf, torch.nan])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dt", [FL, BF])
def test_outputs(name, bad, norm, dt):
    x, _, _ = inputs(dt)
    if not norm:
        x["k"] *= K ** -0.5
    want = gated_delta_rule(**x, output_final_state=True, qk_l2norm=norm)
    got = gated_delta_rule(**spoil(x, name, bad), output_final_state=True, qk_l2norm=norm)
    for a, b, m in zip(want, got, reach(name)):
        assert torch.equal(a[~m], b[~m])
        assert not torch.isfinite(b[m]).any()


@pytest.mark.parametrize("dt", [FL, BF])
def test_a_padded_batch(dt):
    """What lies behind a sequence in its row may be anything."""
    x, _, _ = inputs(dt)
    lens = [130, 7]
    for n in ("q", "k", "v", "g", "beta"):
        for b, m in enumerate(lens):
            x[n][b, m:] = 0
    want, _ = gated_delta_rule(**x, qk_l2norm=True)
    for n, bad in zip(("q", "k", "v", "g", "beta"), (torch.nan, torch.inf, -torch.inf, torch.nan,
                                                     torch.inf)):
        for b, m in enumerate(lens):
            x[n][b, m:] = bad
    o, _ = gated_delta_rule(**x, qk_l2norm=True)
    for b, m in enumerate(lens):
        assert torch.equal(o[b, :m], want[b, :m])


@pytest.mark.parametrize("name", ["k", "v", "g", "beta"])
@pytest.mark.parametrize("at", [0, 63, 64, 700, 1099])
@pytest.mark.parametrize("dt", [FL, BF])
def test_segments(name, at, dt):
    """The same where a sequence is cut into segments that run in parallel."""
    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)   # noqa: E731
    T = 1100
    x = dict(q=r(1, T, 1, 100).to(dt), k=r(1, T, 1, 100).to(dt), v=r(1, T, 1, 40).to(dt),
             g=-0.01 * r(1, T, 1).abs(), beta=torch.sigmoid(r(1, T, 1)))
    want, _ = gated_delta_rule(**x, qk_l2norm=True)
    x[name][(0, at, 0, COL)[:x[name].dim()]] = torch.nan
    got, ht = gated_delta_rule(**x, qk_l2norm=True, output_final_state=True)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[:, at:, :, slice(COL, COL + 1) if name == "v" else slice(None)] = True
    assert torch.equal(got[~bad], want[~bad]) and torch.equal(torch.isfinite(got), ~bad)
    assert torch.equal(torch.isfinite(ht), ~bad[:, -1, :, None].expand_as(ht))


@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta", "do", "dht"])
@pytest.mark.parametrize("bad", [torch.inf, torch.nan])
@pytest.mark.parametrize("dt", [FL, BF])
def test_gradients_of_others(name, bad, dt):
    """Other batch rows and the heads of other keys have the same gradients, to the bit."""
    x, do, dht = inputs(dt)

    def run(x, do, dht):
        x = {n: t.clone().requires_grad_() for n, t in x.items()}
        outs = gated_delta_rule(**x, output_final_state=True, qk_l2norm=True)
        return dict(zip(x, torch.autograd.grad(outs, list(x.values()), [do, dht])))

    want = run(x, do, dht)
    if name == "do":
        do[ROW, AT, 2 * HEAD, COL] = bad
    elif name == "dht":
        dht[ROW, 2 * HEAD, 3, COL] = bad
    else:
        x = spoil(x, name, bad)
    got = run(x, do, dht)
    for n, b in got.items():
        a, heads = want[n], HEAD if n in "qk" else slice(2 * HEAD, 2 * HEAD + 2)
        m = torch.zeros(a.shape, dtype=torch.bool, device=DEV)
        if n == "initial_state":
            m[ROW, heads] = True
        else:
            m[ROW, :, heads] = True
        assert torch.equal(a[~m], b[~m]), n
    assert not all(torch.isfinite(b).all() for b in got.values())
