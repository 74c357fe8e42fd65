"""Segments where a block has 64 columns, and of packed sequences that fill the device by themselves."""

import importlib

import pytest
import torch

dmod = importlib.import_module("tops.ops.delta.gated_delta_rule")
BF = torch.bfloat16


@pytest.mark.parametrize("B,chunks,HV,K,V,L", [
    (1, 128, 8, 256, 256, 16), (1, 128, 8, 128, 256, 8), (2, 64, 8, 200, 256, 16),
    (4, 32, 8, 129, 256, 16), (4, 32, 8, 128, 256, 8), (8, 32, 8, 256, 256, 1 << 20)])
def test_keys_of_more_than_128(B, chunks, HV, K, V, L):
    """The second pass has a block for each of 256 CUs at most, unless L is least for the fold."""
    c = dmod._Chunks(B, 64 * chunks, None, BF, HV, K, V, None)
    assert c.L == L and c.nsegs == B * max(1, -(-chunks // L))
    if L < chunks:
        assert c.nsegs * HV * -(-V // (128 if K <= 128 else 64)) <= 256


def test_packed_sequences_that_fill_the_device():
    f, counts = dmod._segment, [28, 5, 33, 2, 47, 1, 8, 9]
    assert f(counts, 16) == 11    # half of it: all segments at once
    assert f(counts, 32) == 17    # more: by the average
    assert f([30, 40, 50], 64) == 50 and f([30, 40, 50], 32) == 17


@pytest.mark.gpu
@pytest.mark.parametrize("K,V", [(256, 40), (129, 90)])
@pytest.mark.parametrize("lens", [[1100], [700, 20, 0, 500]])
@pytest.mark.parametrize("dt", [torch.float32, BF])
def test_wide_keys_in_segments(lens, K, V, dt):
    import test_gpu_delta as t

    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x, r = t.make(1, cu[-1], 1, 2, K, V, dt, S=len(lens), norm=True)
    x["g"] *= 0.05   # what is before a segment has to matter at its end
    t.check(x, r, cu=cu if len(lens) > 1 else None, norm=True)
