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
    some 95 powers of two above what a thread of each wave reads first (wave w's ids
    are 3072 w .. and its first part half of them); temperatures at which a power in
    32 bits is off by most, short of it and past it."""
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
        x[r, 3072 * 2 + 40 + r] = float(low[i])
        x[r, 3072 * 3 + 1900] = x[r, 3072 * 9 + 1700 + r] = float(high[i])
    return x, torch.rand(2 * count, generator=g), torch.from_numpy(t[pick])


@pytest.mark.parametrize("top_p,kept", [(0.5, 1), (0.5 + 2.0 ** -24, 2)])
def test_the_largest_logits_past_the_first_part(top_p, kept):
    """Half of the mass is the first's, exactly; a step of p more is not."""
    x, u, t = late_rows(24)
    check(x, u, t, top_p=top_p)
    probs = torch.empty_like(x, device="cuda")
    ops.sample(x.cuda(), u.cuda(), t.cuda(), top_p=top_p, probs=probs)
    assert (probs > 0).sum(1).tolist() == [kept] * 48
