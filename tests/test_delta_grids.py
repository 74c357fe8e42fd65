"""Sizes whose launches would have 2^32 threads or more are refused before anything runs."""

import pytest

from test_delta_refusals import DELTA, PTRS, entry

LONG = dict(DELTA, HV=1, V=8, K=8, seg_chunks=1 << 20)


def sizes(chunks, C=64):
    return dict(LONG, T=chunks * C, chunks=chunks, nsegs=-(-chunks // (1 << 20)))


@pytest.mark.parametrize("name,train", [("tops_gla_delta_bwd", 0), ("tops_gla_delta_bwd", 1),
                                        ("tops_gla_delta_fwd", 1)])
@pytest.mark.parametrize("dtype,C,most", [(1, 64, 1 << 23), (0, 32, 1 << 24)])
def test_gradients(name, train, dtype, C, most):
    """A block a chunk and head of 512 threads in bfloat16, 256 in float32; a forward whose backward
    would not fit is refused too."""
    for chunks, code, what in ((most, 2, "grid"), (most - 1, 1, "NULL")):
        rc, msg = entry(name, "tops_gla_delta_args",
                        **{**sizes(chunks, C), "dtype": dtype, "train": train})
        assert rc == code and what in msg, (chunks, msg)


def test_forward_alone():
    for chunks, code, what in ((1 << 24, 2, "grid"), ((1 << 24) - 1, 1, "NULL")):
        rc, msg = entry("tops_gla_delta_fwd", "tops_gla_delta_args", **sizes(chunks))
        assert rc == code and what in msg, (chunks, msg)


@pytest.mark.parametrize("K,threads", [(256, 512), (128, 256), (64, 128)])
def test_fold(K, threads):
    """A block for 16 columns of each head and sequence, of two threads a padded key."""
    V = 16 * 512
    most = (1 << 32) // (512 * threads)
    for nseq, code, what in ((most, 2, "grid"), (most - 1, 1, "NULL")):
        rc, msg = entry("tops_gla_delta_fwd", "tops_gla_delta_args", **{
            **DELTA, "HV": 1, "K": K, "V": V, "T": 64 * 2 * nseq, "seqs": 64, "nseq": nseq,
            "chunks": 2 * nseq, "nsegs": nseq + 1, "seg_chunks": 2})
        assert rc == code and what in msg, (nseq, msg)


def test_no_fold_without_segments():
    rc, msg = entry("tops_gla_delta_fwd", "tops_gla_delta_args", **{
        **DELTA, **PTRS, "HV": 1, "K": 256, "V": 8192, "T": 1 << 20, "seqs": 64, "nseq": 1 << 14,
        "chunks": 1 << 14, "nsegs": 1 << 14, "seg_chunks": 2})
    assert rc == 1 and "keep" in msg, msg
