"""The example model with its block of the gated delta rule behind a layer norm: packed prompts and
served tokens against the whole forward, and a few training steps.

Bounds, float32: as of the model without the block, 1e-3 of the logits' size (order 1). The block
adds sums of 256 products of values of order 1 and a recurrence of 40 tokens that keeps its state
bounded (keys of length 1, 0 < beta < 1), whose two orders differ by some 2^-24 times the square root
of these counts, below 1e-4."""

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
    return HybridLM(delta=True).to(DEV)


def test_served_tokens_equal_the_whole_forward():
    m = model()
    gen = torch.Generator().manual_seed(4)
    seqs = [torch.randint(0, 64, (n,), generator=gen).tolist() for n in (80, 8, 40)]
    cuts = [73, 1, 33]
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
    assert not any(p[[1, 3]].any() for p in pools[2])


def test_gradients_are_differences():
    """Along a random direction of all of the block's parameters, in float32: the loss is a mean of
    order 1 with a relative error of some 1e-6, so that differences over a step of 1e-2 have an
    absolute one of 2e-4 beside the step's own of the third order (a few 1e-4 of a slope of order
    0.1 for a direction of length 1)."""
    m = model()
    gen = torch.Generator().manual_seed(5)
    x = torch.randint(0, 64, (4, 70), generator=gen).to(DEV)
    loss = lambda: torch.nn.functional.cross_entropy(   # noqa: E731
        m(x[:, :-1])[0].flatten(0, 1), x[:, 1:].flatten())
    params = list(m.delta.parameters())
    grads = torch.autograd.grad(loss(), params)
    assert all(torch.isfinite(g).all() and g.any() for g in grads)
    total = sum(float((g.double() ** 2).sum()) for g in grads) ** 0.5
    ways = [g / total for g in grads]   # the steepest direction: a slope of `total`
    ends = []
    with torch.no_grad():
        for step in (1e-2, -2e-2):
            for p, w in zip(params, ways):
                p += step * w
            ends.append(float(loss()))
    slope = (ends[0] - ends[1]) / 2e-2
    assert abs(slope - total) < 1e-3 + 0.02 * total, (slope, total)


def test_training_runs():
    from hybrid_lm import generate, train

    m = model()
    train(m, 3, DEV, report=lambda s: None)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    assert generate(m, [[5, 6, 0], [7, 0]], 4).shape == (2, 4)
