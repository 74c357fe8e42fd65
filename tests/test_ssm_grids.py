"""Sizes whose launch would have 2^32 threads or more are refused before any HIP call; the largest
ones below are not (they fail here on the next check, a missing pointer)."""

import pytest

from test_ssm_refusals import entry

SCAN = dict(T=1, D=4096, N=16, G=1, piece=64, dtype=1)
PTRS = dict.fromkeys(("dy", "du", "ddelta", "dB", "dC", "chunk_h"), 64)


@pytest.mark.parametrize("batch,fits", [((1 << 20) - 1, True), (1 << 20, False)])
def test_scan(batch, fits):
    rc, msg = entry("tops_gla_selective_scan_fwd", "tops_gla_scan_args", batch=batch, nseq=batch,
                    **SCAN)
    assert (rc, "A must" in msg if fits else "grid" in msg) == (1 if fits else 2, True), msg


# 512 threads for 64 channels of 64 states
@pytest.mark.parametrize("batch,fits", [((1 << 17) - 1, True), (1 << 17, False)])
def test_scan_bwd(batch, fits):
    rc, msg = entry("tops_gla_selective_scan_bwd", "tops_gla_scan_args", batch=batch, nseq=batch,
                    **{**SCAN, "N": 64}, **PTRS)
    assert (rc, "A must" in msg if fits else "grid" in msg) == (1 if fits else 2, True), msg


# a block has 256 / 4 channels of two rows
@pytest.mark.parametrize("batch,fits", [((1 << 19) - 2, True), (1 << 19, False)])
def test_scan_step(batch, fits):
    rc, msg = entry("tops_gla_selective_scan_step", "tops_gla_scan_step_args", batch=batch,
                    slots=batch, D=4096, N=16, G=1, dtype=1)
    assert (rc, "NULL" in msg if fits else "grid" in msg) == (1 if fits else 2, True), msg


# a block has 4 rows of final states of 256 channels
@pytest.mark.parametrize("batch,fits", [((1 << 20) - (1 << 13), True), (1 << 20, False)])
def test_conv(batch, fits):
    rc, msg = entry("tops_gla_causal_conv_fwd", "tops_gla_conv_args", batch=batch, nseq=batch, T=1,
                    D=4096, W=4, dtype=1)
    assert (rc, "w must" in msg if fits else "grid" in msg) == (1 if fits else 2, True), msg


@pytest.mark.parametrize("batch,fits", [((1 << 20) - 1, True), (1 << 20, False)])
def test_conv_step(batch, fits):
    rc, msg = entry("tops_gla_causal_conv_step", "tops_gla_conv_step_args", batch=batch,
                    slots=batch, D=4096, W=4, dtype=1)
    assert (rc, "NULL" in msg if fits else "grid" in msg) == (1 if fits else 2, True), msg


# more than 256 heads: a token a block
@pytest.mark.parametrize("batch,fits", [((1 << 24) - 1, True), (1 << 24, False)])
def test_qk(batch, fits):
    rc, msg = entry("tops_gla_qk_norm_rope_fwd", "tops_gla_qk_args", batch=batch, T=1, Hq=600, Hk=1,
                    D=8, dtype=1, eps=1e-6)
    assert (rc, "NULL" in msg if fits else "grid" in msg) == (1 if fits else 2, True), msg
