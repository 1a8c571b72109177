"""How linear_fp8 rounds: once, to nearest even, with what is added inside that
rounding, and with sums that lose no more than documented.

The matrix unit drops what lies more than 13 bits below the largest of eight
products.  Cut towards zero, consecutive eights, normal operands in 8 bits: 2.1e-5
of the results' size (rms, from that arithmetic in 64 bits, for groups' scales
alike or 2^8 apart); what the fp32 sums add is below it (2^-24 of the size for
each of at most 70 instructions in a chain, at random).

Two consequences that a wrong rounding does not have:

- With the exact product's own bf16 rounding r taken away inside the rounding,
  out = bf16(sum - r) is the sum's loss plus the rest v - r that r left, both of
  which bf16 holds to 2^-8 of them: |v - r| <= 2^-8 |v|, so out is off v - r by
  2.1e-5 and 2^-8 2^-8 = 1.5e-5 of the size at most (rms: 2.6e-5 together, as
  they are independent; 2^-15 = 3.05e-5 asked for).  A product rounded before the
  subtraction gives zeros, off by the rounding itself, 1.7e-3.
- A result is the exact value's nearest bf16 value unless a border between two
  lies within the loss: of the same arithmetic's results 98.3% are (97% asked
  for), and the others are the value beside it.  Cut results are it half of the
  time."""
import pytest
import torch

from specdec import ops
from test_gpu_fp8_large import operand, values

pytestmark = pytest.mark.gpu

# few rows: one to four row tiles, scales read directly and by way of LDS (7168 <
# K <= 31744 inputs, more than 4 rows), K up to chains of 70 instructions; then the
# four tiles (rows and features of a workgroup, steps of rows it holds)
CALLS = [(1, 2048, 4096, None), (5, 576, 3000, None), (4, 8192, 2048, None), (5, 8192, 2048, None),
         (15, 7300, 4001, None), (40, 8192, 2048, None), (60, 5000, 3001, None), (33, 31700, 1000, None),
         (64, 8192, 4096, None), (90, 70000, 300, None), (70, 700, 16001, (64, 128, 4)),
         (1000, 520, 2100, (128, 128, 4)), (900, 4200, 2333, (128, 128, 4)), (1000, 600, 4500, (128, 128, 3)),
         (2048, 4225, 8000, (256, 256, 3))]


def ordered(v):
    """bf16 values as integers, neighbouring values one apart."""
    i = v.view(torch.int16).int()
    return torch.where(i < 0, -(i & 0x7FFF), i)


@pytest.mark.parametrize("rows,k,n,tile", CALLS)
def test_one_rounding_to_nearest(rows, k, n, tile):
    block = ops.linear_fp8_block(rows, -(-k // 128) * 128, n)
    assert block == tile if tile else block[2] == 0
    x, xs = operand(rows, k, rows + k)
    wc, ws = operand(n, k, n, 0.05)
    w = ops.tile_weight_fp8(wc)
    v = values(x, xs) @ values(wc, ws).t().contiguous()
    nearest = v.to(torch.bfloat16)

    got = ops.linear_fp8(x, xs, w, ws)
    same = (got == nearest).double().mean().item()
    assert same >= 0.97, same
    sized = v.abs() > 0.05 * v.norm() / v.numel() ** 0.5  # a bf16 step there is above the loss
    assert int((ordered(got) - ordered(nearest)).abs()[sized].max()) <= 1

    rest = v - nearest.double()
    for out in (None, -nearest):
        left = ops.linear_fp8(x, xs, w, ws, out=out, add=-nearest if out is None else out)
        off = ((left.double() - rest).norm() / v.norm()).item()
        assert off <= 2.0 ** -15, off
