"""Sequences of one token, whose distance to a next one says nothing."""

import importlib

import pytest
import torch

from test_delta_refusals import DELTA, PTRS, entry
from tops.ops.delta import gated_delta_rule

dmod = importlib.import_module("tops.ops.delta.gated_delta_rule")


@pytest.mark.parametrize("name", ["q_st", "k_st", "v_st", "do_st"])
@pytest.mark.parametrize("st", [1 << 24, -1, 1 << 40])
@pytest.mark.parametrize("T,code,what", [(1, 1, "keep"), (2, 2, "2^24")])
def test_entry(name, st, T, code, what):
    """With one token it goes on to the next check, the workspace's."""
    rc, msg = entry("tops_gla_delta_bwd", "tops_gla_delta_args",
                    **{**DELTA, **PTRS, "T": T, name: st})
    assert rc == code and what in msg, msg


def test_tokens_are_not_copied():
    t = torch.zeros(3 * 2 * 8, dtype=torch.bfloat16).as_strided((3, 1, 2, 8), (16, 1 << 25, 8, 1))
    assert dmod._tokens(t, t.dtype) is t
    t = torch.empty((1 << 25) + 1, dtype=torch.bfloat16).as_strided((1, 2, 1, 1), (0, 1 << 25, 1, 1))
    assert dmod._tokens(t, t.dtype).stride(1) == 1   # two tokens are


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_one_token_of_a_token_major_batch(dt):
    """[T, B, heads, columns] of 2^25 elements a token, of which one token is there."""
    dev = "cuda:0"
    gen = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)   # noqa: E731
    B, H, HV, K, V = 3, 2, 4, 64, 40
    d = dict(q=r(B, 1, H, K).to(dt), k=r(B, 1, H, K).to(dt), v=r(B, 1, HV, V).to(dt))
    far = {n: t.as_strided(t.shape, (t.stride(0), 1 << 25, *t.stride()[2:])) for n, t in d.items()}
    rest = dict(g=-r(B, 1, HV).abs(), beta=torch.sigmoid(r(B, 1, HV)),
                initial_state=r(B, HV, K, V))
    up = r(B, 1, HV, V).to(dt)
    runs = []
    for x, u in ((d, up), (far, up.as_strided(up.shape, (HV * V, 1 << 25, V, 1)))):
        x = {n: t.detach().requires_grad_() for n, t in {**x, **rest}.items()}
        o, ht = gated_delta_rule(**x, output_final_state=True, qk_l2norm=True)
        runs.append([o, ht, *torch.autograd.grad([o, ht], list(x.values()),
                                                 [u, torch.ones_like(ht)])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
