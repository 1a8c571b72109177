"""Sizes that the 8-bit operators refuse because a launch cannot hold them (no
GPU needed: each call returns before any launch)."""
import pytest

from specdec import _lib

EUNSUPPORTED, BF16, F32 = 3, 2, 0
FAKE = 1 << 20  # never dereferenced


# lanes of a row: 64 up to a width of 512, twice as many with each doubling, 1024 from 4097 on
@pytest.mark.parametrize("dim,lanes", [(1, 64), (512, 64), (513, 128), (1025, 256), (2049, 512), (4097, 1024),
                                       (8193, 1024), (16384, 1024)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_refuses_more_lanes_than_a_launch_holds(dim, lanes, dtype):
    """A launch holds fewer than 2^32 lanes, in workgroups of at least 256."""
    norm = _lib.load().specdec_add_rmsnorm_fp8
    for rows in (((1 << 32) - max(lanes, 256)) // lanes + 1, (1 << 32) // lanes, (1 << 32) // lanes + 1, 1 << 31, 1 << 40):
        assert norm(FAKE, None, FAKE, None, dtype, rows, dim, 1e-5, FAKE, FAKE, None) == EUNSUPPORTED, rows
        assert norm(FAKE, FAKE, FAKE, FAKE, dtype, rows, dim, 1e-5, FAKE, FAKE, None) == EUNSUPPORTED, rows
