"""How exact the gated delta rule is where its inputs are bfloat16: nothing on the way is less exact
than two bfloat16 parts, states are as exact as float32 sums, and results are rounded once.

Bounds, in the 2-norm. A value in two bfloat16 parts is off by 2^-17 of itself at most (half a step of
a remainder that is half a step, 2^-8 of the value's power of two). A float32 sum of n terms has n
roundings of 2^-24, which are independent: sqrt(n) of them. A result of several such operands is, before
its own rounding, off by d: their number times 2^-17 and three such sums one after another, twice, as
the two terms of a result may cancel by half. Rounded, it then differs from the rounded exact value
where a border lies between the two, of all values a share of d / step, by a step each: sqrt(d step) of
the whole, step = 2^-7."""

import pytest
import torch

from delta_ref import F64, delta, sum_roundings
from tops.ops.delta import gated_delta_rule

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FL = torch.bfloat16, torch.float32
STEP = 2.0 ** -7          # of bfloat16
TWO_PARTS = 2.0 ** -17
# operands in two parts on the way to a result:
#   o: the state, the scores, the written values;  dq: the written values, the state, the scores'
#   gradient;  dk: the written values, the right side's gradient, both states, two gradients of scores;
#   dv: the right side's gradient;  dbeta: that, the state, the written values, the system's gradient;
#   dg: all of dq's, dk's and dbeta's, as differences of sums
PARTS = {"o": 3, "q": 3, "k": 6, "v": 1, "beta": 4, "g": 13}
NAMES = ("q", "k", "v", "g", "beta", "initial_state")

CASES = [(1, 40, 1, 1, 64, 64, None), (2, 200, 1, 2, 128, 128, None), (1, 130, 2, 2, 200, 40, None),
         (1, 1100, 1, 2, 64, 96, None), (1, 900, 1, 2, 128, 64, [0, 30, 700, 700, 900]),
         (1, 1100, 1, 1, 256, 40, None), (1, 1000, 1, 2, 200, 130, [0, 620, 1000])]


def make(B, T, H, HV, K, V, cu, gdt):
    gen = torch.Generator().manual_seed(T + K)
    r = lambda *s: torch.randn(*s, generator=gen)   # noqa: E731
    S = B if cu is None else len(cu) - 1
    x = dict(q=r(B, T, H, K).to(BF), k=r(B, T, H, K).to(BF), v=r(B, T, HV, V).to(BF),
             g=(-0.1 * r(B, T, HV).abs()).to(gdt), beta=torch.sigmoid(r(B, T, HV)).to(gdt),
             initial_state=r(S, HV, K, V) * K ** -0.5)
    return x, r(B, T, HV, V).to(BF), r(S, HV, K, V)


def sums(K, T):
    return sum_roundings(K, T) ** 0.5 * 2.0 ** -24


def inside(name, K, T):
    return 2 * (PARTS[name] * TWO_PARTS + 3 * sums(K, T))


def off(got, want):
    got, want = got.detach().cpu().to(F64), want.detach().to(F64)
    return ((got - want).norm() / want.norm()).item()


def rounded_once(name, got, want, K, T):
    """got is the rounded want, but for values next to a border."""
    e, most = off(got, want.detach().to(BF)), (inside(name, K, T) * STEP) ** 0.5
    assert e <= most, f"{name}: {e:.3g} off the rounded value, {most:.3g} allowed"


def run(x, cu, to=lambda t: t.to(DEV)):
    d = {n: to(t).detach().requires_grad_() for n, t in x.items()}
    return d, gated_delta_rule(**d, output_final_state=True, cu_seqlens=cu, qk_l2norm=True)


def oracle(x, cu):
    c = {n: t.to(F64).requires_grad_() for n, t in x.items()}
    return c, delta(*(c[n] for n in NAMES), cu=cu, l2norm=True)


@pytest.mark.parametrize("B,T,H,HV,K,V,cu", CASES)
def test_outputs_are_rounded_once(B, T, H, HV, K, V, cu):
    x, _, _ = make(B, T, H, HV, K, V, cu, FL)
    _, (o, _) = run(x, cu)
    _, (want, _) = oracle(x, cu)
    rounded_once("o", o, want, K, T)


@pytest.mark.parametrize("B,T,H,HV,K,V,cu", CASES)
def test_states_are_float32(B, T, H, HV, K, V, cu):
    """Final states: two sums, the values and the state, of such sums; gradients of initial ones: of
    both passes."""
    x, do, dh = make(B, T, H, HV, K, V, cu, FL)
    d, (o, ht) = run(x, cu)
    c, (ro, rht) = oracle(x, cu)
    e = off(ht, rht)
    assert e <= 2 ** 0.5 * sums(K, T), f"ht: {e:.3g} off, {2 ** 0.5 * sums(K, T):.3g} allowed"
    got, = torch.autograd.grad([o, ht], [d["initial_state"]], [do.to(DEV), dh.to(DEV)])
    want, = torch.autograd.grad([ro, rht], [c["initial_state"]], [do.to(F64), dh.to(F64)])
    e = off(got, want)
    assert e <= 2 * sums(K, T), f"dh0: {e:.3g} off, {2 * sums(K, T):.3g} allowed"


@pytest.mark.parametrize("gdt", [FL, BF])
@pytest.mark.parametrize("B,T,H,HV,K,V,cu", CASES)
def test_gradients_are_rounded_once(B, T, H, HV, K, V, cu, gdt):
    x, do, dh = make(B, T, H, HV, K, V, cu, gdt)
    d, outs = run(x, cu)
    c, refs = oracle(x, cu)
    got = torch.autograd.grad(outs, [d[n] for n in NAMES[:5]], [do.to(DEV), dh.to(DEV)])
    want = torch.autograd.grad(refs, [c[n] for n in NAMES[:5]], [do.to(F64), dh.to(F64)])
    for n, t, w in zip(NAMES, got, want):
        if t.dtype is BF:
            rounded_once(n, t, w, K, T)
        else:   # not rounded at all
            e = off(t, w)
            assert e <= inside(n, K, T), f"d{n}: {e:.3g} off, {inside(n, K, T):.3g} allowed"
