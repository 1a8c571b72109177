"""What the 8-bit operators refuse: sizes that a launch cannot hold, and outputs
and addends of another shape than the product's (no GPU needed: each call
returns before any launch)."""
import pytest
import torch

from specdec import _lib, ops

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


def test_a_product_of_rows_of_several_dimensions_takes_an_output_of_its_shape():
    """x [2, 3, Kp]: an out or add [3, 2, N] holds as many rows, in another order."""
    cpu, bf16 = torch.device("cpu"), torch.bfloat16
    lead, rows, n = torch.Size((2, 3)), 6, 5

    def check(t):
        return ops._fp8_output(cpu, t, lead, rows, n, "add")

    good = torch.zeros(2, 3, 5, dtype=bf16)
    wide = torch.zeros(2, 3, 9, dtype=bf16)
    assert check(good) == (good.data_ptr(), 5)
    assert check(good.view(6, 5)) == (good.data_ptr(), 5)  # its rows
    assert check(wide[..., 2:7]) == (wide.data_ptr() + 4, 9)
    for bad in (torch.zeros(3, 2, 5, dtype=bf16), torch.zeros(6, 1, 5, dtype=bf16), torch.zeros(30, dtype=bf16),
                torch.zeros(2, 3, 6, dtype=bf16), torch.zeros((), dtype=bf16), torch.zeros(1, 5, dtype=bf16).expand(6, 5),
                torch.zeros(3, 2, 5, dtype=bf16).transpose(0, 1),  # rows that no one stride reaches
                torch.zeros(2, 5, 3, dtype=bf16).transpose(1, 2)):
        with pytest.raises(ValueError, match="add must be"):
            check(bad)
    one = torch.zeros(5, dtype=bf16)
    assert ops._fp8_output(cpu, one, torch.Size(()), 1, 5, "out") == (one.data_ptr(), 5)
    with pytest.raises(ValueError, match="out must be"):
        ops._fp8_output(cpu, one[:4], torch.Size(()), 1, 5, "out")
    none = torch.zeros(2, 0, 5, dtype=bf16)
    assert ops._fp8_output(cpu, none, torch.Size((2, 0)), 0, 5, "out")[1] == 5


def test_the_choice_of_a_workgroup():
    """On 256 compute units: the tiles that test_gpu_fp8_tiles relies on, and blocks of few rows."""
    from test_gpu_fp8_tiles import CALLS

    def block(rows, k, n, **kw):
        return ops.linear_fp8_block(rows, -(-k // 128) * 128, n, compute_units=256, **kw)

    for tile, call in CALLS:
        assert block(*call) == tile, call
    assert block(1, 576, 960) == (16, 16, 0)
    assert block(5, 2048, 16384) == (16, 32, 0)
    assert block(40, 2048, 16384) == (48, 64, 0)
    assert block(64, 2048, 16384) == (64, 64, 0)
    assert block(288, 2048, 6144) == (64, 128, 4)
    assert block(4096, 2048, 16384) == (256, 256, 3)
    # rows too far apart for a tile's 32-bit offsets are left to the few-row kernel
    assert block(4096, 2048, 16384, x_stride=1 << 25)[2] == 0


def test_the_choice_refuses_what_the_product_refuses():
    assert ops.linear_fp8_block(1048560, 128, 16, compute_units=256)
    for bad in ((-1, 256, 16), (2, 200, 16), (2, 0, 16), (2, 256, 0)):
        with pytest.raises(ops.KernelError):
            ops.linear_fp8_block(*bad, compute_units=256)
    with pytest.raises(ops.KernelError):
        ops.linear_fp8_block(2, 256, 16, x_stride=128, compute_units=256)
    with pytest.raises(ops.KernelError):
        ops.linear_fp8_block(2, 256, 16, compute_units=-1)
    for far in ((1048561, 256, 16), (2, (1 << 23) + 128, 16), (2, 256, (1 << 24) + 1)):
        with pytest.raises(NotImplementedError):
            ops.linear_fp8_block(*far, compute_units=256)
    with pytest.raises(NotImplementedError):
        ops.linear_fp8_block(2, 256, 16, x_stride=(1 << 25) + 16, compute_units=256)
