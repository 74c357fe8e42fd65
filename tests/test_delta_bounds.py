"""What the bounds of tests/test_gpu_delta_accuracy.py rest on: floats in two and in three bfloat16
parts, each the rounded remainder of those before it."""

import torch


def remainders(x):
    """What one, two and three parts leave off."""
    out = []
    for _ in range(3):
        x = x - x.to(torch.bfloat16).float()
        out.append(x)
    return out


def test_parts_of_floats():
    """All floats of [1, 2): two parts are up to 2^-17 off, three hold them exactly."""
    x = torch.arange(1 << 23, dtype=torch.int32).add_(0x3F800000).view(torch.float32)
    one, two, three = remainders(x)
    assert one.abs().max() == 2.0 ** -8
    worst = (two.abs() / x).max().item()
    assert 2.0 ** -18 < worst <= 2.0 ** -17
    assert not three.any()
    assert not remainders(torch.randn(1 << 20) * 2.0 ** torch.randint(-60, 60, (1 << 20,)))[2].any()
