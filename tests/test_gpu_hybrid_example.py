"""The example model: serving token by token against the whole forward, and a few training steps.

Bounds, float32: the served logits come from the same formulas in another order. Sums of up to 512
products of values of order 1 in float32 give relative errors of a few 2^-24 times the square root
of their count; three blocks of them and a recurrence of 40 tokens stay below 1e-3 of the logits'
size (order 1) by more than a factor of ten."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def model():
    from hybrid_lm import HybridLM

    torch.manual_seed(0)
    return HybridLM().to(DEV)


def test_served_tokens_equal_the_whole_forward():
    m = model()
    gen = torch.Generator().manual_seed(3)
    seqs = [torch.randint(0, 64, (n,), generator=gen).tolist() for n in (40, 31, 27)]
    cuts = [33, 1, 20]
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=DEV)
    pools = m.empty_pools(5)
    got = [m.prefill([s[:c] for s, c in zip(seqs, cuts)], pools, slots)]
    for i in range(7):
        token = torch.tensor([s[c + i] for s, c in zip(seqs, cuts)], device=DEV)
        pos = torch.tensor([c + i for c in cuts], device=DEV)
        got.append(m.step(token, pos, pools, slots))
    for b, (s, c) in enumerate(zip(seqs, cuts)):
        with torch.no_grad():
            want = m(torch.tensor([s], device=DEV))[0][0]
        for i, g in enumerate(got):
            torch.testing.assert_close(g[b], want[c - 1 + i], atol=1e-3, rtol=1e-3)


def test_training_learns():
    from hybrid_lm import generate, train

    m = model()
    losses = train(m, 40, DEV, report=lambda s: None)
    first, last = torch.stack(losses[:5]).mean().item(), torch.stack(losses[-5:]).mean().item()
    assert last < first - 0.05, (first, last)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    assert generate(m, [[5, 6, 0], [7, 0]], 4).shape == (2, 4)
