"""linear_fp8 at the sizes its tiles are made for, and 8-bit operators over
tensors past 2^31 elements.  Products against fp64 on the GPU, with the bound of
test_gpu_fp8 taken over all products (the largest of eight is at most their
sum): half a bf16 step of the exact value plus 7 * 2^-13 + (K / 8 + 16) * 2^-23
of sum |x w|."""
import pytest
import torch

from specdec import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
G = 128


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def operand(rows, k, seed, spread=1.0):
    """Rows in 8 bits whose groups' scales differ by up to 2^8, and their values in fp64."""
    g = gen(seed)
    x = spread * torch.randn(rows, k, generator=g, device=DEV)
    x *= torch.exp2(torch.randint(-4, 4, (rows, -(-k // G)), generator=g, device=DEV).float()).repeat_interleave(
        G, dim=1)[:, :k]
    codes, scales = ops.quantize_fp8(x)
    return codes, scales


def values(codes, scales):
    return codes.double() * scales.double().repeat_interleave(G, dim=1)[:, :codes.shape[1]]


def check(got, xv, wv, add=None):
    exact = xv @ wv.t().contiguous()
    lost = (7 * 2.0 ** -13 + (xv.shape[1] / 8 + 16) * 2.0 ** -23) * (xv.abs() @ wv.abs().t().contiguous())
    if add is not None:
        exact = exact + add.double()
        lost = lost + 2.0 ** -24 * exact.abs()
    half = torch.exp2(torch.floor(torch.log2((exact.abs() + lost).clamp_min(1e-30))) - 8)
    err = (got.double() - exact).abs()
    assert bool((err <= half + lost).all()), (err - half - lost).max().item()
    # what one part in a hundred of the products left out would pass
    rms = (got.double() - exact).norm() / exact.norm()
    assert rms.item() < 2.0 ** -8 + 1e-3, rms.item()


# on 256 compute units: the 64 x 128, 128 x 128 (deep, paired) and 256 x 256
# tiles, each whole, ragged in rows and features, and with as few steps as a tile
# can have; widths that end inside a group, inside four and inside sixteen
SHAPES = [(128, 2048, 2816), (100, 1300, 3001), (97, 100, 5000), (1000, 520, 2100), (1024, 2300, 2048),
          (900, 4200, 2333), (1000, 600, 4500), (1500, 2048, 4096), (1792, 128, 8192), (1990, 600, 8170),
          (2048, 2048, 8192), (2048, 4225, 8000)]


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_tiles(rows, k, n, add):
    x, xs = operand(rows, k, rows + k)
    wc, ws = operand(n, k, n, 0.05)
    base = torch.randn(rows, n, generator=gen(1), device=DEV).to(torch.bfloat16) if add else None
    out = torch.full((rows + 2, n), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.linear_fp8(x, xs, ops.tile_weight_fp8(wc), ws, out=out[1:-1], add=base)
    check(out[1:-1], values(x, xs), values(wc, ws), base)
    assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all())


# Few rows: each block of 16 x 16, 16 x 32, 16 x 64, 32 x 64, 48 x 64 and 64 x 64
# (on 256 compute units), rows and features that end inside it, with scales read
# from memory (up to 7168 inputs, and past 31744) and by way of LDS, and up to 4 rows
FEW = [(16, 1000), (11, 5000), (15, 16001), (30, 16001), (41, 16001), (60, 16001), (120, 2039), (170, 2039), (4, 1000)]


@pytest.mark.parametrize("k", [600, 5000, 7300, 8192])
@pytest.mark.parametrize("rows,n", FEW)
def test_blocks_of_few_rows(rows, n, k):
    x, xs = operand(rows, k, rows + k)
    wc, ws = operand(n, k, n, 0.05)
    w = ops.tile_weight_fp8(wc)
    base = torch.randn(rows, n, generator=gen(1), device=DEV).to(torch.bfloat16)
    out = torch.full((rows + 2, n), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.linear_fp8(x, xs, w, ws, out=out[1:-1], add=base)
    check(out[1:-1], values(x, xs), values(wc, ws), base)
    assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all())
    if rows <= 64:  # however many rows, and so whichever block and way of the scales
        for m in (1, 4, 5, 17, 33):
            if m < rows:
                assert torch.equal(ops.linear_fp8(x[:m], xs[:m], w, ws, add=base[:m]), out[1:1 + m]), m


@pytest.mark.parametrize("rows,k,n", [(5, 31700, 100), (60, 31700, 16001), (5, 31800, 100), (60, 31800, 3001), (90, 70000, 100)])
def test_long_rows(rows, k, n):
    x, xs = operand(rows, k, rows + k)
    wc, ws = operand(n, k, n, 0.05)
    check(ops.linear_fp8(x, xs, ops.tile_weight_fp8(wc), ws), values(x, xs), values(wc, ws))


def test_tiles_repeat_their_bits():
    """The same call again, alone and among others on a second stream: the same bits."""
    for rows, k, n in ((100, 1300, 3001), (1000, 520, 2100), (1000, 600, 4500), (1990, 600, 8170)):
        x, xs = operand(rows, k, 3)
        wc, ws = operand(n, k, 4, 0.05)
        w = ops.tile_weight_fp8(wc)
        first = ops.linear_fp8(x, xs, w, ws)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        outs = []
        for _ in range(4):
            outs.append(ops.linear_fp8(x, xs, w, ws))
            with torch.cuda.stream(side):
                outs.append(ops.linear_fp8(x, xs, w, ws))
        torch.cuda.synchronize()
        assert all(torch.equal(o, first) for o in outs)


def test_output_past_two_to_the_31_elements():
    rows, k, n = 33000, 256, 66000
    x, xs = operand(rows, k, 5)
    wc, ws = operand(n, k, 6, 0.05)
    out = ops.linear_fp8(x, xs, ops.tile_weight_fp8(wc), ws)
    wv = values(wc, ws)
    for lo in (0, 16384, 32536, 32984):  # the last two behind 2^31
        pick = slice(lo, lo + 16)
        check(out[pick], values(x[pick], xs[pick]), wv)


def test_rows_past_two_to_the_31_codes():
    rows, k, n = 280000, 8192, 24
    x, xs = operand(64, k, 7)
    x = x.view(torch.uint8).repeat(rows // 64 + 1, 1)[:rows].view(torch.float8_e4m3fn)
    xs = xs.view(torch.uint8).repeat(rows // 64 + 1, 1)[:rows].view(torch.float8_e8m0fnu)
    wc, ws = operand(n, k, 8, 0.05)
    out = ops.linear_fp8(x, xs, ops.tile_weight_fp8(wc), ws)
    assert torch.equal(out, out[:64].repeat(rows // 64 + 1, 1)[:rows])
    check(out[-16:], values(x[-16:], xs[-16:]), values(wc, ws))


def test_rows_to_8_bits_past_two_to_the_31_elements():
    rows, k = 1050000, 2048
    x = torch.randn(rows, k, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(k, dtype=torch.bfloat16, device=DEV)
    tail = x[-5:].clone()
    for f in (ops.quantize_fp8, ops.silu_mul_fp8, lambda v: ops.add_rmsnorm_fp8(v, None, w, 1e-5)):
        codes, scales = f(x)
        c, s = f(tail)
        assert torch.equal(codes[-5:].view(torch.uint8), c.view(torch.uint8))
        assert torch.equal(scales[-5:].view(torch.uint8), s.view(torch.uint8))
        del codes, scales
