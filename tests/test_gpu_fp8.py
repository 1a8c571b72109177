"""The 8-bit projections' operators -- rows to 8 bits with a scale for each
128 values, RMSNorm with the residual addition and SiLU(gate) * up written in
that format, and the product of 8-bit rows and an 8-bit weight -- against
their definitions in 64 bits.

The conversion itself is exact in the inputs' types, so codes and scales are
compared bit for bit.  The norm and the activation reach the rounding through
a few fp32 operations: with a relative error eps of the value, a code stands
for the value to half an e4m3 step plus eps |y|, and a scale may differ only
where the group's maximum lies within eps of a power of two times 448.  A
product's tolerance is the bf16 rounding's half step plus what the matrix unit
loses: among eight products it drops what lies more than 13 bits below the
largest one's exponent (so less than 2^-13 of the largest, of each of the seven
others; the largest itself has 8 bits), and the sums of eight are added in fp32,
each sum within a unit (2^-23)."""
import pytest
import torch

from specdec import ops

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
G = 128
TYPES = [torch.bfloat16, torch.float32]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ref_scale_exponents(y):
    """e of each group of y [R, K] fp64: [R, ceil(K / 128)]."""
    r, k = y.shape
    groups = -(-k // G)
    pad = torch.zeros(r, groups * G, dtype=torch.float64)
    pad[:, :k] = torch.where(y.isfinite(), y, torch.zeros_like(y))
    amax = pad.view(r, groups, G).abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(amax > 0, e, torch.full_like(e, -126)).clamp_min(-126), amax


def ref_codes(y, e):
    """Values of the codes of y [R, K] fp64 under exponents e: [R, Kp]."""
    r, k = y.shape
    v = torch.zeros(r, e.shape[1] * G, dtype=torch.float64)
    v[:, :k] = y
    v = v / torch.exp2(e.double()).repeat_interleave(G, dim=1)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    q = torch.round(v / step) * step  # to even
    return torch.where(v.isfinite(), q, torch.full_like(q, float("nan")))


def shapes_ok(codes, scales, rows, k):
    assert codes.dtype == torch.float8_e4m3fn and tuple(codes.shape) == (rows, -(-k // G) * G)
    assert scales.dtype == torch.float8_e8m0fnu and tuple(scales.shape) == (rows, -(-k // 512) * 4)
    groups = -(-k // G)
    assert bool((scales.view(torch.uint8)[:, groups:] == 127).all())  # ones
    assert bool((codes.view(torch.uint8)[:, k:] == 0).all())  # zeros


def check_exact(codes, scales, y):
    """Codes and scales of y, bit for bit (NaN codes of either sign)."""
    rows, k = y.shape
    codes, scales = codes.cpu(), scales.cpu()
    shapes_ok(codes, scales, rows, k)
    e, _ = ref_scale_exponents(y)
    assert torch.equal(scales.view(torch.uint8)[:, :e.shape[1]].int(), e.int() + 127)
    want, got = ref_codes(y, e), codes.double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def check_near(codes, scales, y, eps, tiny=0.0):
    """Codes and scales of values within eps |y| + tiny of y (fp64)."""
    rows, k = y.shape
    codes, scales = codes.cpu(), scales.cpu()
    shapes_ok(codes, scales, rows, k)
    e, amax = ref_scale_exponents(y)
    got_e = scales.view(torch.uint8)[:, :e.shape[1]].int() - 127
    slack = amax * eps + (tiny if isinstance(tiny, float) else tiny.amax())
    lo, _ = ref_scale_exponents_of(amax - slack)
    hi, _ = ref_scale_exponents_of(amax + slack)
    assert bool(((got_e >= lo) & (got_e <= hi)).all())
    s = torch.exp2(got_e.double()).repeat_interleave(G, dim=1)[:, :k]
    got = codes.double()[:, :k] * s
    assert torch.equal(got.isnan(), ~y.isfinite())
    fine = y.isfinite()
    half = torch.exp2(torch.floor(torch.log2(((y.abs() * (1 + eps)) / s).clamp_min(2.0 ** -6))) - 4) * s
    err = torch.where(fine, (got - y).abs() - half - eps * y.abs() - tiny, torch.full_like(y, -1.0))
    assert err.max().item() <= 0, err.max().item()


def ref_scale_exponents_of(amax):
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(amax > 0, e, torch.full_like(e, -126)).clamp_min(-126), amax


# ------------------------------------------------------------------ quantize --
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 127), (1, 128), (2, 129), (3, 511), (5, 512), (4, 513), (7, 576),
                                    (1, 2048), (33, 2051), (2, 8192), (300, 40), (3, 20000)])
def test_quantize_is_exact(dtype, rows, k):
    g = gen(rows * 31 + k)
    x = (torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, k), generator=g).float())).to(dtype)
    codes, scales = ops.quantize_fp8(x.to(DEV))
    check_exact(codes, scales, x.double())


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_borders(dtype):
    """Maxima at, just below and just above 448 2^e, ties, zeros, the smallest
    and largest values of the type, negative zeros."""
    big = torch.finfo(dtype).max
    small = torch.finfo(dtype).smallest_normal
    rows = []
    for m in (448.0, 450.0, 447.0, 448.0 * 2 ** 20, 450.0 * 2 ** -20, 512.0, 0.875, 0.8789, 1.0, big, small, small / 64, 0.0):
        row = torch.zeros(256, dtype=torch.float64)
        row[5] = -m
        # every tie between two codes near the maximum, and among the subnormals
        row[10:100] = m * (torch.arange(90, dtype=torch.float64) + 0.5) / 256
        row[100:120] = m / 448 * 2.0 ** -10 * torch.arange(20, dtype=torch.float64)
        row[200] = m / 3
        rows.append(row)
    x = torch.stack(rows).to(dtype)
    x[0, 130] = -0.0
    codes, scales = ops.quantize_fp8(x.to(DEV))
    check_exact(codes, scales, x.double())


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_infinities_and_nan_keep_to_themselves(dtype):
    x = torch.randn(4, 300, generator=gen(2)).to(dtype)
    x[0, 3], x[1, 130], x[1, 131], x[2, 299] = float("nan"), float("inf"), float("-inf"), float("nan")
    x[3, :128] = float("inf")  # nothing finite in the group
    codes, scales = ops.quantize_fp8(x.to(DEV))
    check_exact(codes, scales, x.double())
    clean = x.clone()
    clean[~clean.isfinite()] = 0
    c2, s2 = ops.quantize_fp8(clean.to(DEV))
    assert torch.equal(scales.view(torch.uint8), s2.view(torch.uint8))
    same = x.isfinite().to(DEV)
    assert torch.equal(codes.view(torch.uint8)[:, :300][same], c2.view(torch.uint8)[:, :300][same])


def test_quantize_strides_and_shapes():
    x = torch.randn(6, 5, 700, generator=gen(3)).to(torch.bfloat16).to(DEV)
    for view in (x[:, 2], x[:, :, 3:600], x[1, 1, 7:], x.transpose(0, 1), x[..., :64].transpose(1, 2),
                 x[:1, 0].expand(9, 700), x[::2, ::2, 1::2]):
        codes, scales = ops.quantize_fp8(view)
        assert codes.shape[:-1] == view.shape[:-1] and scales.shape[:-1] == view.shape[:-1]
        k = view.shape[-1]
        check_exact(codes.view(-1, codes.shape[-1]), scales.view(-1, scales.shape[-1]),
                    view.cpu().double().reshape(-1, k))


def test_outputs_given_are_written_and_nothing_else():
    x = torch.randn(3, 200, generator=gen(4)).to(DEV)
    raw_c = torch.full((5, 256), 77, dtype=torch.uint8, device=DEV)
    raw_s = torch.full((5, 4), 99, dtype=torch.uint8, device=DEV)
    c, s = raw_c[1:4].view(torch.float8_e4m3fn), raw_s[1:4].view(torch.float8_e8m0fnu)
    got = ops.quantize_fp8(x, c, s)
    assert got[0] is c and got[1] is s
    check_exact(c, s, x.cpu().double())
    for raw, mark in ((raw_c, 77), (raw_s, 99)):
        assert bool((raw[0] == mark).all()) and bool((raw[4] == mark).all())


def test_no_rows():
    for shape in ((0, 300), (2, 0, 300)):
        x = torch.zeros(*shape, device=DEV)
        codes, scales = ops.quantize_fp8(x)
        assert tuple(codes.shape) == (*shape[:-1], 384) and tuple(scales.shape) == (*shape[:-1], 4)
        assert tuple(ops.silu_mul_fp8(x)[0].shape) == (*shape[:-1], 256)
        assert tuple(ops.add_rmsnorm_fp8(x, None, torch.ones(300, device=DEV), 1e-5)[0].shape) == (*shape[:-1], 384)
        w, ws = weight(torch.randn(20, 300, generator=gen(1)))
        assert tuple(ops.linear_fp8(codes, scales, w, ws).shape) == (*shape[:-1], 20)


# ------------------------------------------------------------------ the norm --
# The sum of squares: a chain of at most 64 squares and sums in a thread, six
# additions in the wave, four of the waves; half of its relative error reaches
# the root; then the quotient, the sum with eps, the root (one unit, 2^-23) and
# two products: (64 + 1 + 10) / 2 + 1 / 2 + 1 / 2 + 2 + 2 < 48 half units.
NORM_EPS = 48 * 2.0 ** -24


def norm_ref(h, weight, eps):
    x = h.double()
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("rows,dim", [(1, 1), (2, 63), (1, 128), (5, 200), (32, 576), (1, 2048), (300, 2048), (3, 2049),
                                      (2, 4100), (3, 8192), (2, 8200), (1, 16384)])
def test_add_rmsnorm(dtype, delta, rows, dim):
    g = gen(rows * 13 + dim)
    hidden = (torch.randn(rows, dim, generator=g) * torch.exp(torch.randn(dim, generator=g))).to(dtype)
    d = (0.3 * torch.randn(rows, dim, generator=g)).to(dtype) if delta else None
    w = (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype)
    h = hidden if d is None else (hidden.float() + d.float()).to(dtype)
    y = norm_ref(h, w, 1e-5)
    hd = hidden.to(DEV)
    codes, scales = ops.add_rmsnorm_fp8(hd, None if d is None else d.to(DEV), w.to(DEV), 1e-5)
    assert torch.equal(hd.cpu(), h)  # in place
    check_near(codes, scales, y, NORM_EPS)
    if delta:  # the sum elsewhere: the same bits, hidden left alone
        hd, out = hidden.to(DEV), torch.full((rows, dim), 5.0, dtype=dtype, device=DEV)
        c2, s2 = ops.add_rmsnorm_fp8(hd, d.to(DEV), w.to(DEV), 1e-5, summed=out)
        assert torch.equal(hd.cpu(), hidden) and torch.equal(out.cpu(), h)
        assert torch.equal(c2.view(torch.uint8), codes.view(torch.uint8))
        assert torch.equal(s2.view(torch.uint8), scales.view(torch.uint8))


def test_add_rmsnorm_zero_rows_and_values_that_are_no_numbers():
    h = torch.randn(4, 300, generator=gen(6))
    h[0] = 0
    h[1, 7] = float("nan")
    h[2, 9] = float("inf")
    w = torch.ones(300)
    codes, scales = ops.add_rmsnorm_fp8(h.to(DEV), None, w.to(DEV), 1e-5)
    v = codes.cpu().double()
    assert bool((v[0] == 0).all())
    assert bool(v[1, :300].isnan().all())  # the row's mean is NaN
    assert bool(v[2, 9].isnan()) and bool((v[2, torch.arange(384) != 9] == 0).all())  # x / inf, inf / inf
    assert bool((v[:, 300:] == 0).all())
    check_near(codes[3:], scales[3:], norm_ref(h[3:], w, 1e-5), NORM_EPS)


def test_rows_do_not_depend_on_the_call():
    h = torch.randn(70, 576, generator=gen(7)).to(torch.bfloat16).to(DEV)
    w = torch.ones(576, dtype=torch.bfloat16, device=DEV)
    gu = torch.randn(70, 1200, generator=gen(8)).to(DEV)
    for f in (lambda r: ops.add_rmsnorm_fp8(h[r].contiguous(), None, w, 1e-5), lambda r: ops.silu_mul_fp8(gu[r])):
        codes, scales = f(slice(None))
        for r in (0, 1, 33, 69):
            c, s = f(slice(r, r + 1))
            assert torch.equal(c.view(torch.uint8), codes[r:r + 1].view(torch.uint8))
            assert torch.equal(s.view(torch.uint8), scales[r:r + 1].view(torch.uint8))


# ------------------------------------------------------------ the activation --
# exp to two units (2^-23 each), then a sum, a quotient and a product
SILU_EPS = 7 * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inter", [(1, 1), (3, 100), (2, 128), (5, 1536), (40, 8192), (7, 1001), (2, 9999)])
def test_silu_mul(dtype, rows, inter):
    g = gen(rows + inter)
    gu = (4 * torch.randn(rows, 2 * inter, generator=g)).to(dtype)
    codes, scales = ops.silu_mul_fp8(gu.to(DEV))
    gate, up = gu.double().split(inter, dim=1)
    # below -126 log 2 e^-gate passes fp32, and gate / inf is 0 where the value is gate e^gate
    check_near(codes, scales, gate / (1 + torch.exp(-gate)) * up, SILU_EPS, tiny=gate.abs() * up.abs() * 2.0 ** -126)


def test_silu_mul_far_gates_and_strided_rows():
    wide = torch.randn(6, 2 * 300 + 50, generator=gen(9))
    wide[0, 10:20] = torch.tensor([-200.0, -100.0, -89.0, -87.0, 87.0, 100.0, 200.0, 3e38, -3e38, 0.0])
    wide[1, 12], wide[2, 310] = float("inf"), float("nan")
    gu = wide[:, 10:610]
    codes, scales = ops.silu_mul_fp8(wide.to(DEV)[:, 10:610])
    gate, up = gu.double().split(300, dim=1)
    y = gate / (1 + torch.exp(-gate)) * up
    y = torch.where(y.abs() > torch.finfo(torch.float32).max, torch.full_like(y, float("inf")), y)
    check_near(codes, scales, y, SILU_EPS, tiny=gate.abs().clamp_max(1e3) * up.abs().nan_to_num(0) * 2.0 ** -126)


# --------------------------------------------------------------- the product --
def weight(w):
    codes, scales = ops.quantize_fp8(w.to(DEV))
    return ops.tile_weight_fp8(codes), scales


def values(codes, scales):
    c = codes.cpu().double()
    return c * scales.cpu().double().repeat_interleave(G, dim=-1)[..., :c.shape[-1]]


def half_step(v):
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(1e-30))) - 8)


def check_product(got, xv, wv, add=None):
    """got [R, N] against xv [R, Kp] wv [N, Kp]^T (fp64 values of the codes)."""
    exact = xv @ wv.t()
    lost = torch.zeros_like(exact)
    for lo in range(0, xv.shape[1], 8):  # seven of eight products cut at 2^-13 of the largest
        p = (xv[:, None, lo:lo + 8] * wv[None, :, lo:lo + 8]).abs().amax(-1)
        lost += 7 * 2.0 ** -13 * p
    mag = xv.abs() @ wv.abs().t()
    lost += (xv.shape[1] / 8 + 16) * 2.0 ** -23 * mag  # the sums of eight, and the waves', in fp32
    if add is not None:
        exact = exact + add.double()
        lost += 2.0 ** -24 * exact.abs()
    err = (got.cpu().double() - exact).abs() - lost
    # the rounding's half step: at the exact value, or one binade up where the loss may carry it there
    bound = half_step(exact.abs() + lost)
    assert bool((err <= bound).all()), (err - bound).max().item()
    # over all values: a rounding is at most 2^-8 of its value, so the norm of the errors
    # is at most 2^-8 of the values' norm plus the norm of the losses; 128 inputs left
    # out, taken twice or scaled by another's scale change it by 1 / sqrt(groups)
    rms = (got.cpu().double() - exact).norm() / exact.norm()
    assert rms.item() <= 2.0 ** -8 + lost.norm() / exact.norm(), rms.item()


def rows_of(rows, k, seed, dtype=torch.float32):
    g = gen(seed)
    # scales that differ from group to group and from row to row
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-6, 6, (rows, -(-k // G)), generator=g).float()
                                                        ).repeat_interleave(G, dim=1)[:, :k]
    return x.to(dtype)


SHAPES = [(1, 1, 1), (1, 128, 16), (1, 576, 960), (5, 100, 33), (5, 2048, 512), (3, 8192, 64), (8, 1536, 576),
          (16, 700, 100), (17, 2048, 128), (33, 640, 200), (64, 1100, 48), (65, 512, 100), (100, 2048, 130),
          (128, 384, 256), (130, 1300, 257), (257, 2048, 144), (300, 576, 529), (513, 256, 300)]


@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_linear_fp8(rows, k, n):
    x, xs = ops.quantize_fp8(rows_of(rows, k, rows + k).to(DEV))
    wc, ws = ops.quantize_fp8(0.05 * rows_of(n, k, n).to(DEV))
    got = ops.linear_fp8(x, xs, ops.tile_weight_fp8(wc), ws)
    assert got.shape == (rows, n) and got.dtype == torch.bfloat16
    check_product(got, values(x, xs), values(wc, ws))


@pytest.mark.parametrize("rows,k,n", [(1, 576, 576), (5, 2048, 200), (40, 1536, 100), (70, 600, 257), (260, 512, 130)])
def test_linear_fp8_adds_before_the_rounding(rows, k, n):
    x, xs = ops.quantize_fp8(rows_of(rows, k, 1).to(DEV))
    wc, ws = ops.quantize_fp8(0.05 * rows_of(n, k, 2).to(DEV))
    w = ops.tile_weight_fp8(wc)
    base = (3 * torch.randn(rows, n, generator=gen(3))).to(torch.bfloat16)
    got = ops.linear_fp8(x, xs, w, ws, add=base.to(DEV))
    check_product(got, values(x, xs), values(wc, ws), base)
    out = base.to(DEV)
    assert ops.linear_fp8(x, xs, w, ws, out=out, add=out) is out  # in place: the same bits
    assert torch.equal(out, got)


@pytest.mark.parametrize("rows,k,n", [(64, 2048, 300), (40, 8192, 100), (30, 576, 960), (64, 128, 64)])
def test_linear_fp8_rows_do_not_depend_on_the_other_rows(rows, k, n):
    x, xs = ops.quantize_fp8(rows_of(rows, k, 5).to(DEV))
    w, ws = weight(0.05 * rows_of(n, k, 6))
    together = ops.linear_fp8(x, xs, w, ws)
    for r in range(rows):
        assert torch.equal(ops.linear_fp8(x[r:r + 1], xs[r:r + 1], w, ws), together[r:r + 1]), r
    for m in (2, 5, 8, 9, 16, 17, 31, 32, 33, 48, 49):
        if m <= rows:
            assert torch.equal(ops.linear_fp8(x[:m], xs[:m], w, ws), together[:m]), m


@pytest.mark.parametrize("rows", [4, 90, 300])
def test_linear_fp8_strided_operands(rows):
    """Rows out of wider tensors and every third row; out and add column blocks
    of wider tensors at odd offsets, whose neighbours are left alone."""
    k, n = 700, 161
    xc, xsc = ops.quantize_fp8(rows_of(3 * rows, k, 8).to(DEV))
    wc, ws = ops.quantize_fp8(0.05 * rows_of(n, k, 9).to(DEV))
    w = ops.tile_weight_fp8(wc)
    x, xs = xc[::3], xsc[::3]
    out = torch.full((rows, n + 20), 7.0, dtype=torch.bfloat16, device=DEV)
    addw = torch.randn(rows, n + 9, generator=gen(10)).to(torch.bfloat16).to(DEV)
    ops.linear_fp8(x, xs, w, ws, out=out[:, 3:3 + n], add=addw[:, 5:5 + n])
    assert torch.equal(out[:, 3:3 + n], ops.linear_fp8(x.contiguous(), xs.contiguous(), w, ws,
                                                       add=addw[:, 5:5 + n].contiguous()))
    check_product(out[:, 3:3 + n], values(x, xs), values(wc, ws), addw[:, 5:5 + n].cpu())
    assert bool((out[:, :3] == 7).all()) and bool((out[:, 3 + n:] == 7).all())
    three = ops.linear_fp8(xc.view(rows, 3, -1), xsc.view(rows, 3, -1), w, ws)
    assert three.shape == (rows, 3, n)


def test_linear_fp8_rows_far_apart():
    """Rows 2^26 bytes apart (their offsets pass 32 bits) are copied first; 2^25
    are read in place."""
    w, ws = weight(0.05 * rows_of(40, 128, 1))
    x, xs = ops.quantize_fp8(rows_of(70, 128, 2).to(DEV))
    want = ops.linear_fp8(x, xs, w, ws)
    for log in (25, 26):
        far = torch.empty((69 << log) + 128, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
        view = far.as_strided((70, 128), (1 << log, 1))
        view.copy_(x)
        assert torch.equal(ops.linear_fp8(view, xs, w, ws), want)
        assert torch.equal(ops.linear_fp8(view[:64], xs[:64], w, ws), ops.linear_fp8(x[:64], xs[:64], w, ws))
        del far, view


@pytest.mark.parametrize("rows", [3, 80, 300])
def test_linear_fp8_carries_nan(rows):
    """A NaN in a row makes that row NaN and no other; one in a weight's row that feature."""
    x = rows_of(rows, 300, 11)
    x[1, 17] = float("nan")
    w = 0.05 * rows_of(70, 300, 12)
    w[69, 299] = float("inf")
    xc, xs = ops.quantize_fp8(x.to(DEV))
    wt, ws = weight(w)
    got = ops.linear_fp8(xc, xs, wt, ws).cpu()
    want = torch.zeros(rows, 70, dtype=torch.bool)
    want[1], want[:, 69] = True, True
    assert torch.equal(got.isnan(), want)


def test_scales_at_the_ends_of_the_range():
    """Groups near 2^-126 and near 2^119: the product's scale is their sum."""
    x, w = torch.randn(5, 256, generator=gen(13)), torch.randn(40, 256, generator=gen(14))
    for up, down in ((2.0 ** 100, 2.0 ** -100), (2.0 ** -110, 2.0 ** 100), (2.0 ** 60, 2.0 ** 50), (2.0 ** -60, 2.0 ** -50)):
        xc, xs = ops.quantize_fp8((x * up).to(DEV))
        wc, ws = ops.quantize_fp8((w * down).to(DEV))
        got = ops.linear_fp8(xc, xs, ops.tile_weight_fp8(wc), ws)
        check_product(got, values(xc, xs), values(wc, ws))


# ------------------------------------------------- together, streams, graphs --
def mlp(x, delta, ln, gu, down, resid=None):
    """The MLP half of a decoder layer over 8-bit projections."""
    h = x.clone()
    c, s = ops.add_rmsnorm_fp8(h, delta, ln, 1e-5)
    a = ops.linear_fp8(c, s, *gu)
    c, s = ops.silu_mul_fp8(a)
    return ops.linear_fp8(c, s, *down, out=h, add=h)


def mlp_parts(dim, inter, seed):
    g = gen(seed)
    gu, down = 0.05 * torch.randn(2 * inter, dim, generator=g), 0.05 * torch.randn(dim, inter, generator=g)
    ln = (1 + 0.1 * torch.randn(dim, generator=g)).to(torch.bfloat16)
    return ln, gu, down


@pytest.mark.parametrize("rows,dim,inter", [(1, 576, 1536), (5, 512, 1000), (100, 576, 640), (300, 256, 1536)])
def test_mlp_of_a_layer(rows, dim, inter):
    """The operators as a layer runs them, against fp64 of the unquantised
    weights: each of the two projections sees operands with at most 2^-4 of
    relative error a side, of random sign, so its relative error is about
    sqrt(2) 2^-4 / sqrt(3) = 5% of its output's size, and below 10% with the
    activation's part."""
    ln, gu, down = mlp_parts(dim, inter, 20)
    x = torch.randn(rows, dim, generator=gen(21)).to(torch.bfloat16)
    d = torch.randn(rows, dim, generator=gen(22)).to(torch.bfloat16)
    got = mlp(x.to(DEV), d.to(DEV), ln.to(DEV), weight(gu), weight(down)).cpu().double()
    h = (x.float() + d.float()).to(torch.bfloat16)
    y = norm_ref(h, ln, 1e-5)
    gate, up = (y @ gu.double().t()).split(inter, dim=1)
    want = gate / (1 + torch.exp(-gate)) * up @ down.double().t()
    rel = ((got - h.double()) - want).norm() / want.norm()
    assert rel.item() < 0.10, rel.item()


@pytest.mark.parametrize("rows", [5, 40, 200])
def test_graph_replays_and_side_streams(rows):
    """Captured once and replayed over new inputs, with the program's own calls
    between the replays; and on a stream of its own: the eager bits."""
    dim, inter = 576, 1536
    ln, gu, down = mlp_parts(dim, inter, 30)
    ln, gu, down = ln.to(DEV), weight(gu), weight(down)
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
    d = torch.zeros_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mlp(x, d, ln, gu, down)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(x, d, ln, gu, down)
    for i in range(4):
        x.copy_(torch.randn(rows, dim, generator=gen(31 + i)))
        d.copy_(torch.randn(rows, dim, generator=gen(41 + i)))
        eager = mlp(x, d, ln, gu, down)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = mlp(x, d, ln, gu, down)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, eager), i


def test_first_call_inside_a_capture():
    """Kernels that need more than 64 KB of LDS, called for the first time while a
    stream is captured (in a process of its own)."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from specdec import ops
cases = []
for rows, k, n in ((64, 8192, 16384), (100, 1300, 3001), (1000, 520, 2100), (1000, 600, 4500), (1990, 600, 8170)):
    x, xs = ops.quantize_fp8(torch.randn(rows, k, device="cuda"))
    wc, ws = ops.quantize_fp8(torch.randn(n, k, device="cuda"))
    cases.append((x, xs, ops.tile_weight_fp8(wc), ws))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = [ops.linear_fp8(*c) for c in cases]
for i in range(3):
    for o in outs:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, ops.linear_fp8(*c)) for o, c in zip(outs, cases)), i
print("captured")
"""
    pkg = Path(__file__).resolve().parents[1] / "speculative-decoder_amd"
    out = subprocess.run([sys.executable, "-c", code], cwd=pkg, capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_refusals():
    x, xs = ops.quantize_fp8(torch.randn(4, 300, device=DEV))
    w, ws = weight(torch.randn(20, 300, generator=gen(1)))
    with pytest.raises(TypeError):
        ops.quantize_fp8(torch.zeros(2, 8, dtype=torch.float16, device=DEV))
    with pytest.raises(ValueError):
        ops.silu_mul_fp8(torch.zeros(2, 7, device=DEV))
    with pytest.raises(NotImplementedError):
        ops.add_rmsnorm_fp8(torch.zeros(1, 16385, device=DEV), None, torch.ones(16385, device=DEV), 1e-5)
    with pytest.raises(ValueError):
        ops.add_rmsnorm_fp8(torch.zeros(4, 8, device=DEV)[:, :4], None, torch.ones(4, device=DEV), 1e-5)
    with pytest.raises(ValueError):
        ops.add_rmsnorm_fp8(torch.zeros(4, 8, device=DEV), None, torch.ones(8, device=DEV), 1e-5,
                            summed=torch.zeros(4, 8, device=DEV))
    with pytest.raises(ValueError):
        ops.linear_fp8(x[:, :256], xs, w, ws)  # another width than the weight's
    with pytest.raises(ValueError):
        ops.linear_fp8(x, xs[:3], w, ws)
    with pytest.raises(ValueError):
        ops.linear_fp8(x, xs, w, ws[:15])  # 15 features are one tile, the weight has two
    with pytest.raises(ValueError):
        ops.linear_fp8(x, xs, w, ws, out=torch.zeros(4, 21, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(TypeError):
        ops.linear_fp8(x, xs, w, ws, add=torch.zeros(4, 20, device=DEV))
    with pytest.raises(ValueError):
        ops.linear_fp8(x, xs, w, ws, out=torch.zeros(1, 20, dtype=torch.bfloat16, device=DEV).expand(4, 20))
