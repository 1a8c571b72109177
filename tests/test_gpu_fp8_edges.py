"""The 8-bit operators where their values or their operands are at an edge:
gates whose SiLU is below fp32's normal values while the product with `up` is
not.  Tolerances as in test_gpu_fp8."""
import pytest
import torch

from specdec import ops
from test_gpu_fp8 import SILU_EPS, TYPES, check_near, gen

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
G = 128

# around the border of the two forms (-80), where 1 / (1 + e^-g) turns subnormal
# (-126 log 2 = -87.34), where e^-g passes fp32 (-128 log 2 = -88.72), where g e^g
# times the largest up falls below the least code (2^-136, near -188), and past it
GATES = [-60.0, -79.5, -79.99999, -80.0, -80.00001, -80.5, -87.0, -87.3, -87.4, -88.0, -88.5, -88.6, -88.7, -88.8,
         -89.0, -92.0, -95.0, -100.0, -103.9, -110.0, -130.0, -150.0, -170.0, -174.0, -180.0, -185.0, -187.0, -190.0,
         -200.0, -1000.0, -3e38]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most", [1.0, 1e10, 1e20, 1e30, 3e38])
def test_silu_of_far_gates_times_large_values(dtype, most):
    """A group of 128 for each gate, so that a group's scale is its values'.  A
    value below fp32's normal ones is within half of fp32's least step, 2^-150,
    and another for the product before it."""
    g = gen(int(torch.tensor(most).log2()))
    gate = torch.tensor(GATES).repeat_interleave(G).repeat(3, 1)
    gate[1] *= 1 + 1e-3 * torch.rand(gate.shape[1], generator=g)
    gate[2, ::2] = torch.randn(gate.shape[1] // 2, generator=g)  # near and far gates in one thread's values
    gate = gate.clamp_min(-3e38)
    up = most * (0.25 + 0.75 * torch.rand(gate.shape, generator=g)) * (1 - 2.0 * (torch.rand(gate.shape, generator=g) < 0.5))
    gu = torch.cat([gate, up], dim=1).to(dtype)
    codes, scales = ops.silu_mul_fp8(gu.to(DEV))
    gate, up = gu.double().split(gate.shape[1], dim=1)
    y = gate / (1 + torch.exp(-gate)) * up
    # a near gate's product with 3e38 can pass fp32's largest value: an infinity there
    y = torch.where(y.abs() > torch.finfo(torch.float32).max, y.sign() * float("inf"), y)
    check_near(codes, scales, y, SILU_EPS, tiny=2.0 ** -149)


def test_silu_of_infinite_gates_and_values():
    """-inf gives -inf / inf = NaN and +inf an infinity, both NaN codes, beside far gates too."""
    inf, nan = float("inf"), float("nan")
    gate = torch.full((2, 256), -100.0)
    gate[1] = 1.0
    up = torch.full((2, 256), 1e30)
    gate[:, 0], gate[:, 1], gate[:, 2], gate[:, 3] = -inf, inf, nan, -nan
    up[:, 4], up[:, 5], up[:, 6] = inf, -inf, nan
    codes, scales = ops.silu_mul_fp8(torch.cat([gate, up], dim=1).to(DEV))
    g, u = gate.double(), up.double()
    check_near(codes, scales, g / (1 + torch.exp(-g)) * u, SILU_EPS, tiny=2.0 ** -149)


def test_norm_of_the_most_rows_a_call_takes():
    rows, dim = (1 << 26) - 4, 16
    h = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
    h[-9:] = torch.randn(9, dim, generator=gen(1)).to(torch.bfloat16)
    h[:3] = torch.randn(3, dim, generator=gen(2)).to(torch.bfloat16)
    w = torch.ones(dim, dtype=torch.bfloat16, device=DEV)
    codes, scales = ops.add_rmsnorm_fp8(h, None, w, 1e-5)
    for part in (slice(0, 5), slice(rows - 12, rows)):
        c, s = ops.add_rmsnorm_fp8(h[part].contiguous(), None, w, 1e-5)
        assert torch.equal(codes[part].view(torch.uint8), c.view(torch.uint8))
        assert torch.equal(scales[part].view(torch.uint8), s.view(torch.uint8))
    with pytest.raises(NotImplementedError):
        ops.add_rmsnorm_fp8(torch.zeros(rows + 1, dim, dtype=torch.bfloat16, device=DEV), None, w, 1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 77), (5, 512), (7, 1003), (40, 2048), (3, 4099), (2, 8192), (5, 8203),
                                      (3, 16384)])
def test_norm_writes_the_sum_over_delta(dtype, rows, dim):
    """summed may be delta, or hidden, itself: the same bits as elsewhere."""
    g = gen(rows + dim)
    hidden, delta = (torch.randn(rows, dim, generator=g).to(dtype).to(DEV) for _ in range(2))
    w = (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).to(DEV)
    summed = torch.empty_like(hidden)
    codes, scales = ops.add_rmsnorm_fp8(hidden, delta, w, 1e-5, summed=summed)
    assert torch.equal(summed, (hidden.float() + delta.float()).to(dtype))
    over = delta.clone()
    before = hidden.clone()
    c, s = ops.add_rmsnorm_fp8(hidden, over, w, 1e-5, summed=over)
    assert torch.equal(over, summed) and torch.equal(hidden, before)
    assert torch.equal(c.view(torch.uint8), codes.view(torch.uint8))
    assert torch.equal(s.view(torch.uint8), scales.view(torch.uint8))
    c, s = ops.add_rmsnorm_fp8(before, delta, w, 1e-5, summed=before)
    assert torch.equal(before, summed)
    assert torch.equal(c.view(torch.uint8), codes.view(torch.uint8))
    assert torch.equal(s.view(torch.uint8), scales.view(torch.uint8))


@pytest.mark.parametrize("rows", [(2, 3), (20, 50)])
def test_product_of_rows_of_two_dimensions_and_its_outputs(rows):
    """out and add of the product's shape, or of its rows; the same rows in
    another arrangement are refused."""
    k, n = 200, 40
    x, xs = ops.quantize_fp8(torch.randn(*rows, k, generator=gen(1)).to(DEV))
    codes, ws = ops.quantize_fp8(torch.randn(n, k, generator=gen(2)).to(DEV))
    w = ops.tile_weight_fp8(codes)
    add = torch.randn(*rows, n, generator=gen(3)).to(torch.bfloat16).to(DEV)
    want = ops.linear_fp8(x.view(-1, x.shape[-1]), xs.view(-1, xs.shape[-1]), w, ws, add=add.view(-1, n))
    out = torch.zeros(*rows, n, dtype=torch.bfloat16, device=DEV)
    assert ops.linear_fp8(x, xs, w, ws, out=out, add=add) is out and torch.equal(out.view(-1, n), want)
    flat = torch.zeros(rows[0] * rows[1], n, dtype=torch.bfloat16, device=DEV)
    ops.linear_fp8(x, xs, w, ws, out=flat, add=add.view(-1, n))
    assert torch.equal(flat, want)
    turned = torch.zeros(rows[1], rows[0], n, dtype=torch.bfloat16, device=DEV)
    for bad in ({"add": turned}, {"out": turned}, {"add": turned.transpose(0, 1)}, {"out": turned.transpose(0, 1)}):
        with pytest.raises(ValueError):
            ops.linear_fp8(x, xs, w, ws, **bad)
