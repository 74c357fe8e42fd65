"""Infinities in the selective state space operators, against the recurrence in 64 bits: where that
is finite the result has the bound of the finite tests, where it is an infinity it is the same
infinity, and a NaN only where the formula has one (inf - inf, 0 * inf).

The other values are positive (A negative), so that an infinity's effects all have one sign and the
recurrence keeps it an infinity almost everywhere."""

import pytest
import torch

import test_gpu_ssm_scan as scan_tests
from ssm_ref import close
from tops.ops.ssm import selective_scan, selective_scan_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")


def make(B, T, D, N, z=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: 0.5 + torch.rand(*s, generator=gen)   # noqa: E731
    x = dict(u=r(B, T, D), delta=0.2 * r(B, T, D), A=-0.2 * r(D, N), B=r(B, T, N), C=r(B, T, N),
             D=r(D), z=r(B, T, D) if z else None, delta_bias=0.1 * r(D),
             initial_state=r(B, D, N))
    return x, r


def same(name, got, ref, mag, terms):
    got = got.detach().cpu()
    ok = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{name}: NaN in other places"
    odd = ~ok & ~torch.isnan(ref)
    assert torch.equal(got[odd].double(), ref[odd]), f"{name}: other infinities"
    close(name, got[ok], ref[ok], mag[ok], terms)


@pytest.mark.parametrize("N", [12, 16])
@pytest.mark.parametrize("softplus", [True, False])
def test_infinite_decay_of_no_step(N, softplus):
    """A of -inf: a token with delta' = 0 leaves the state as it is, any other forgets it, the same
    in the scan and in its single-token form."""
    x, _ = make(3, 1, 20, N)
    x["A"][:, 0] = -INF
    x["delta"][:] = -INF if softplus else 0.0
    x["delta_bias"] = torch.zeros(20)
    x["delta"][2] = 0.25
    ref, mag = scan_tests.reference(dict(x, A=x["A"].double().clamp(min=-1e300)), softplus, None)
    d = {n: t.to(DEV) for n, t in x.items()}
    y, ht = selective_scan(**d, delta_softplus=softplus, output_final_state=True)
    same("y", y, ref["y"], mag["y"], 68)
    same("ht", ht, ref["ht"], mag["ht"], 68)
    state = d.pop("initial_state")
    y = selective_scan_step(state, **{n: t[:, 0] if n in ("u", "delta", "z", "B", "C") else t
                                      for n, t in d.items()}, delta_softplus=softplus)
    same("y", y, ref["y"][:, 0], mag["y"][:, 0], 68)
    same("state", state, ref["ht"], mag["ht"], 68)


@pytest.mark.parametrize("N", [1, 2, 5, 12, 13, 16, 33])
def test_infinite_inputs_of_a_step(N):
    x, r = make(6, 1, 40, N)
    x["u"][1, 0, 3], x["u"][2, 0, 39], x["u"][5, 0, 0] = INF, -INF, INF
    x["delta"][3, 0, 7] = INF
    ref, mag = scan_tests.reference(x, False, None)
    state = x.pop("initial_state").to(DEV)
    y = selective_scan_step(state, **{n: t[:, 0].to(DEV) if n in ("u", "delta", "z", "B", "C")
                                      else t.to(DEV) for n, t in x.items()})
    same("y", y, ref["y"][:, 0], mag["y"][:, 0], 68)
    same("state", state, ref["ht"], mag["ht"], 68)


def check(x, r, dy=None, dht=None):
    d = {n: None if t is None else t.to(DEV).requires_grad_() for n, t in x.items()}
    y, ht = selective_scan(**d, output_final_state=True)
    dy = r(*y.shape) if dy is None else dy
    dht = r(*ht.shape) if dht is None else dht
    names = [n for n, t in d.items() if t is not None]
    got = torch.autograd.grad([y, ht], [d[n] for n in names], [dy.to(DEV), dht.to(DEV)])
    ref, mag = scan_tests.reference(x, False, None, dy, dht)
    B, T, D = x["u"].shape
    terms = 4 * T + 64
    same("y", y, ref["y"], mag["y"], terms)
    same("ht", ht, ref["ht"], mag["ht"], terms)
    for n, t in zip(names, got):
        same("d" + n, t, ref["d" + n], mag["d" + n], terms + B * T + D)


def infinite_inputs(N, T, z):
    """An infinity in the first, a middle and the last token of a sequence."""
    x, r = make(3, T, 70, N, z)
    for b, (t, v) in enumerate(((0, INF), (T // 2, -INF), (T - 1, INF))):
        x["u"][b, t, 3 * b] = x["u"][b, t, 69 - b] = v
    return x, r


# a last tile that is full and one that is not; one piece and several
@pytest.mark.parametrize("N", [8, 16, 32])
@pytest.mark.parametrize("T", [13, 37, 40, 150])
@pytest.mark.parametrize("z", [True, False])
def test_infinite_inputs(N, T, z):
    check(*infinite_inputs(N, T, z))


def infinite_inputs(N, T, z):
    """An infinity in the first, a middle and the last token of a sequence."""
    x, r = make(3, T, 70, N, z)
    for b, (t, v) in enumerate(((0, INF), (T // 2, -INF), (T - 1, INF))):
        x["u"][b, t, 3 * b] = x["u"][b, t, 69 - b] = v
    return x, r


# a last tile that is full and one that is not; one piece and several
@pytest.mark.parametrize("N", [8, 16, 32])
@pytest.mark.parametrize("T", [13, 37, 40, 150])
@pytest.mark.parametrize("z", [True, False])
def test_infinite_inputs(N, T, z):
    check(*infinite_inputs(N, T, z))


def infinite_gradients(N, T):
    """An infinite gradient of the first, a middle and the last token's output."""
    x, r = make(3, T, 70, N)
    dy = r(3, T, 70)
    for b, t in enumerate((0, T // 2, T - 1)):
        dy[b, t, 3 * b] = INF
    return x, r, dy


@pytest.mark.parametrize("N", [8, 16])
@pytest.mark.parametrize("T", [13, 150])
def test_infinite_gradients(N, T):
    check(*infinite_gradients(N, T))


@pytest.mark.parametrize("N", [1, 12, 13, 16])
@pytest.mark.parametrize("T", [13, 150])
def test_infinite_gradient_of_the_final_state(N, T):
    x, r = make(2, T, 70, N)
    dht = r(2, 70, N)
    dht[1, 7, 0] = INF
    check(x, r, None, dht)


@pytest.mark.parametrize("T", [60, 700])
def test_infinite_states_under_strong_decay(T):
    """Each token's decay is far above the smallest number, a piece's product of them is below it:
    an infinite state stays infinite, as it does in the recurrence."""
    x, r = make(2, T, 8, 16, z=False)
    x["A"], x["delta_bias"] = torch.full((8, 16), -20.0), None
    x["delta"] = torch.ones(2, T, 8)
    x["u"][0, 3, 2] = INF
    x["initial_state"][1, 5, 7] = INF
    check(x, r)
    dht = r(2, 8, 16)
    dht[0, 1, 4] = INF
    check(make(2, T, 8, 16, z=False)[0] | {n: x[n] for n in ("A", "delta", "delta_bias")}, r, None,
          dht)


@pytest.mark.parametrize("N", [1, 5, 12, 13, 33])
@pytest.mark.parametrize("T", [13, 37, 40, 150])
@pytest.mark.parametrize("z", [True, False])
def test_infinite_inputs_beside_padded_states(N, T, z):
    check(*infinite_inputs(N, T, z))


@pytest.mark.parametrize("N", [1, 12, 13])
@pytest.mark.parametrize("T", [13, 150])
def test_infinite_gradients_beside_padded_states(N, T):
    check(*infinite_gradients(N, T))


@pytest.mark.parametrize("N", [12, 16])
def test_infinite_steps(N):
    """An infinite delta forgets the state and adds an infinity to it."""
    x, _ = make(2, 45, 70, N)
    x["delta"][0, 20, 3] = x["delta"][1, 44, 69] = INF
    d = {n: t.to(DEV) for n, t in x.items()}
    y, ht = selective_scan(**d, output_final_state=True)
    ref, mag = scan_tests.reference(x, False, None)
    same("y", y, ref["y"], mag["y"], 4 * 45 + 64)
    same("ht", ht, ref["ht"], mag["ht"], 4 * 45 + 64)


@pytest.mark.parametrize("n", ["B", "C"])
@pytest.mark.parametrize("D,N", [(1, 16), (70, 12), (130, 16), (64, 16), (9, 5), (20, 40)])
def test_infinite_rows(n, D, N):
    """A row that all channels read: the lanes without a channel add nothing to its gradient."""
    x, r = make(2, 37, D, N)
    x[n][0, 20, N - 1] = INF
    check(x, r)
