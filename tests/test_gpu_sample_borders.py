"""ops.sample where a cut falls among values that are hard to tell apart:
against the sort in 64 bits, as test_gpu_sample.py."""
import numpy as np
import pytest
import torch

from specdec import ops
from test_gpu_sample import check

pytestmark = pytest.mark.gpu

MOST = torch.finfo(torch.float32).max
CUTS = [dict(top_k=50), dict(top_k=1000), dict(top_p=0.9), dict(top_k=3000, top_p=0.7), dict(top_p=0.9, min_p=0.5)]


def close_rows(vocab, dtype):
    """Rows of thousands of values within 6e-36 of one another, or neighbours among the type's."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.zeros(9, vocab)
    x[0, 7] = 1e-40
    x[1, vocab - 3] = -1e-40
    x[2] = torch.randn(vocab, generator=g) * 1e-37
    x[3] = torch.randn(vocab, generator=g) * 1e-39
    x[4] = torch.randn(vocab, generator=g) * 1e-44
    x[5, :8] = torch.randn(8, generator=g)
    x[5, 8] = 1e-37
    x[6] = torch.where(torch.rand(vocab, generator=g) < 0.5, 1.0, 1.0 + torch.finfo(dtype).eps)
    x[7] = torch.tensor([-MOST, 0.0, 1e-40, 1e-38])[torch.randint(0, 4, (vocab,), generator=g)]
    x[8] = torch.randn(vocab, generator=g) * 1e-37
    x[8, 100:110] = torch.randn(10, generator=g) + 4
    x = x.to(dtype)
    x[7].clamp_(min=torch.finfo(dtype).min)  # the nearest bf16 to -MOST is -inf
    return x, torch.rand(9, generator=g)


@pytest.mark.parametrize("vocab", [3001, 49152])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cut", range(len(CUTS)))
def test_values_that_differ_by_next_to_nothing(cut, dtype, vocab):
    check(*close_rows(vocab, dtype), **CUTS[cut])


@pytest.mark.parametrize("cut", range(len(CUTS)))
def test_close_values_in_more_rows_than_compute_units(cut):
    x, _ = close_rows(3001, torch.float32)
    check(x.repeat(31, 1), torch.rand(279, generator=torch.Generator().manual_seed(3)), **CUTS[cut])


def late_rows(count):
    """(x [2 count, 49152], u, temperatures): two equal logits hold all the weight,
    some 95 powers of two above what each wave reads first (of 16 waves a 16th of the
    ids each, its first part half of them); temperatures at which a power in 32 bits is
    off by most, short of it and past it."""
    wave = 49152 // 16
    rng = np.random.default_rng(0)
    f = np.float32
    t = rng.uniform(0.2, 1.5, 200000).astype(f)
    low = rng.uniform(0, 4, t.size).astype(f)
    c = 1.4426950408889634 / t.astype(np.float64)
    high = (low + rng.uniform(90, 99.5, t.size) / c).astype(f)
    off = (high - low) * c.astype(f) - (high.astype(np.float64) - low) * c
    order = np.argsort(off)
    pick = np.concatenate([order[:count], order[-count:]])
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2 * count, 49152, generator=g) * 0.3 - 5
    for r, i in enumerate(pick):
        x[r, wave * 2 + 40 + r] = float(low[i])
        x[r, wave * 3 + 1900] = x[r, wave * 9 + 1700 + r] = float(high[i])
    return x, torch.rand(2 * count, generator=g), torch.from_numpy(t[pick])


@pytest.mark.parametrize("top_p,kept", [(0.5, 1), (0.5 + 2.0 ** -24, 2)])
def test_the_largest_logits_past_the_first_part(top_p, kept):
    """Half of the mass is the first's, exactly; a step of p more is not."""
    x, u, t = late_rows(24)
    check(x, u, t, top_p=top_p)
    probs = torch.empty_like(x, device="cuda")
    ops.sample(x.cuda(), u.cuda(), t.cuda(), top_p=top_p, probs=probs)
    assert (probs > 0).sum(1).tolist() == [kept] * 48


def check_near(x, u, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """As check, where a cut may lie so near to a border that 64 bits do not tell:
    34 weights of 1 and 33 of e^-34 are 34 or 34 + 6e-14 by the order of their sum,
    and half of that is 17 of them or 18.  Sums of n weights are off by n 2^-53, a
    weight by 1e-13 at most (4e-14 in the kernel and the rounding of its power of at
    most 62 where it counts), so a goal this near to a prefix's mass may be on either
    side of it; the token and the distribution have to be those of the prefix taken."""
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
    temperature, top_p, min_p = f32(temperature), f32(top_p), f32(min_p)
    probs = torch.full(x.shape, 9.0, device="cuda")
    got = ops.sample(x.cuda(), u.cuda(), temperature, top_k, top_p, min_p, probs=probs).cpu()
    probs = probs.cpu().double()
    n = x.shape[1]
    off = 4 * n * 2.0 ** -53 + 1e-13
    for r in range(len(x)):
        ids = torch.argsort(x[r].double(), descending=True, stable=True)
        if top_k:
            ids = ids[:top_k]
        e = x[r].double()[ids]
        w = torch.where(e == e[0], 1.0, torch.exp((e - e[0]) / temperature))
        mass, ends = w.cumsum(0), []
        for side in (-1, 1):
            keep = len(ids)
            if top_p < 1:
                keep = min(keep, int((mass < (top_p + side * off) * mass[-1]).sum()) + 1)
            if min_p > 0:
                keep = min(keep, max(1, int((w >= min_p * (1 - side * off)).sum())))
            ends.append(keep)
        keep = min(max(int((probs[r] > 0).sum()), ends[0]), ends[1])
        p = torch.zeros(n, dtype=torch.float64)
        p[ids[:keep]] = w[:keep] / w[:keep].sum()
        assert torch.equal(probs[r] > 0, p.float() > 0), (r, ends)
        assert bool(((probs[r] - p).abs() <= p * 2.0 ** -23 + 2.0 ** -149).all()), r
        run = p.cumsum(0)
        token = int(((run > float(u[r])) & (p > 0)).nonzero()[0])
        assert int(got[r]) == token or float((run - float(u[r])).abs().min()) < off, (r, int(got[r]), token)


@pytest.mark.parametrize("vocab", [100, 3001])
@pytest.mark.parametrize("kw", [dict(top_p=0.5), dict(top_p=0.9, min_p=0.3), dict(top_k=60, top_p=0.7), dict(min_p=0.6), {}])
@pytest.mark.parametrize("temperature", [1e-45, 1e-40, 1e-39, 1e-37, 1e-32, 1e32, 1e37, 3.3e38])
def test_temperatures_at_the_ends_of_fp32(temperature, kw, vocab):
    """Powers of two that no fp32 product of a difference and 1 / temperature
    holds: rows of one value, of values that weigh alike at this temperature, and of
    values that weigh next to nothing beside the first."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.zeros(5, vocab)
    x[1] = (torch.randn(vocab, generator=g).double() * min(temperature, 1e37)).float()
    x[2] = torch.randn(vocab, generator=g)
    x[3] = torch.tensor([-MOST, 0.0, MOST])[torch.randint(0, 3, (vocab,), generator=g)]
    x[4] = (torch.randint(-3, 1, (vocab,), generator=g).double() * min(temperature, 1e38)).float()
    check_near(x, torch.rand(5, generator=g), temperature, **kw)


@pytest.mark.parametrize("kw", [{}, dict(top_p=0.9), dict(top_k=50, top_p=0.95), dict(top_k=100000, top_p=0.5), dict(min_p=0.01)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_widest_rows(dtype, kw):
    """2^24 ids, and a few fewer from an address that is not aligned."""
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(1, 1 << 24, generator=g) * 1.5).to(dtype)
    u = torch.rand(1, generator=g)
    check(x, u, **kw)
    if not kw:
        got = ops.sample(x.cuda()[:, 3:-2], u.cuda())
        assert int(got) == int(check(x[:, 3:-2].contiguous(), u))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [{}, dict(top_p=0.9), dict(top_k=50, top_p=0.95), dict(top_k=1000), dict(min_p=0.05), dict(temperature=0.0),
                                dict(top_p=0.999, min_p=0.0001)])
def test_vocabularies_that_a_mask_leaves_little_of(kw, dtype):
    """Rows whose first half, all but a few ids, all but the last or all but a stretch are
    -inf, and rows with NaN or the type's lowest value in their place."""
    v = 49152
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(10, v, generator=g) * 2).to(dtype)
    keep = torch.zeros(10, v, dtype=torch.bool)
    keep[0, v // 2:] = keep[6, v // 2:] = keep[8, v // 2:] = True
    keep[1, torch.randperm(v, generator=g)[:40]] = True
    keep[2, -1] = True
    keep[3, 30000:30700] = keep[7, 30000:30700] = keep[9, 30000:30700] = True
    keep[4] = torch.arange(v) % (v // 16) >= v // 32  # nothing in the part that is read first
    keep[5, torch.randperm(v, generator=g)[:3000]] = True
    fill = torch.tensor([float("-inf")] * 6 + [float("nan")] * 2 + [torch.finfo(dtype).min] * 2).to(dtype)
    x = torch.where(keep, x, fill[:, None])
    check(x, torch.rand(10, generator=g), **kw)
