"""ops.sample against a sort in 64 bits: tokens equal, distributions within fp32's rounding."""
import pytest
import torch

from specdec import ops
from tree_ref import draw

pytestmark = pytest.mark.gpu

# A token may differ where u lies this near to its border, relative to the total:
# V weights and sums each within a few steps of 2^-53, and the kernel's total off by as much.
def _gap(v):
    return 8 * v * 2.0 ** -53


def rows_of(seed, rows, vocab, dtype=torch.float32, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * spread
    x[:, ::97] += 4
    return x.to(dtype), torch.rand(rows, generator=g)


def check(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, **kw):
    rows, vocab = x.shape
    per = lambda v, r, f: f(v[r]) if isinstance(v, torch.Tensor) else v
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
    put = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v
    probs = torch.full((rows, vocab), 9.0, device="cuda")
    args = [put(v) for v in (temperature, top_k, top_p, min_p)]
    got = ops.sample(x.cuda(), u.cuda(), *args, probs=probs, **kw).cpu()
    alone = ops.sample(x.cuda(), u.cuda(), *args).cpu()
    assert torch.equal(got, alone)
    probs = probs.cpu().double()
    for r in range(rows):
        want, p, gap = draw(x[r], float(u[r]), f32(per(temperature, r, float)), per(top_k, r, int),
                            f32(per(top_p, r, float)), f32(per(min_p, r, float)))
        assert int(got[r]) == want or gap < _gap(vocab), (r, int(got[r]), want, gap)
        # the kept ids are the same ones; each weight and the total in 64 bits, one rounding to fp32
        assert torch.equal(probs[r] > 0, p.float() > 0), r
        assert bool(((probs[r] - p).abs() <= p * 2.0 ** -23 + 2.0 ** -149).all()), r
    return got


@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 64, 65, 255, 1000, 1023, 1025, 4099, 16384, 49152, 65537, 128001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_whole_softmax(vocab, dtype):
    check(*rows_of(vocab, 3, vocab, dtype), temperature=0.8)


@pytest.mark.parametrize("vocab", [7, 1000, 49152, 100003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top_k", [1, 2, 5, 50, 400, 1000, 5000, 200000])
def test_top_k(vocab, dtype, top_k):
    check(*rows_of(vocab + top_k, 3, vocab, dtype), top_k=top_k)


@pytest.mark.parametrize("spread", [0.01, 1.0, 5.0])
@pytest.mark.parametrize("top_p", [0.0, 1e-6, 0.3, 0.9, 0.95, 0.999, 1.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_p(spread, top_p, dtype):
    """From a few ids to most of the vocabulary."""
    check(*rows_of(7, 2, 20011, dtype, spread), top_p=top_p)


def flat_rows(seed, rows, vocab, dtype, steep):
    """Rows whose nucleus holds thousands of ids: probability falls as rank^-steep."""
    g = torch.Generator().manual_seed(seed)
    rank = torch.stack([torch.randperm(vocab, generator=g) for _ in range(rows)]).float() + 1
    x = 12 - steep * rank.log() + 0.5 * torch.randn(rows, vocab, generator=g)
    return x.to(dtype), torch.rand(rows, generator=g)


@pytest.mark.parametrize("vocab", [16411, 49152, 65537, 128001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steep,kw", [(0.9, dict(top_p=0.9)), (1.0, dict(top_p=0.5, temperature=1.3)),
                                      (0.8, dict(top_p=0.98, min_p=0.0005)), (0.9, dict(top_p=0.7, top_k=6000)),
                                      (1.1, dict(top_p=0.9999))])
def test_wide_nuclei(vocab, dtype, steep, kw):
    check(*flat_rows(vocab, 3, vocab, dtype, steep), **kw)


@pytest.mark.parametrize("vocab,rows", [(1003, 700), (20000, 300), (49152, 270)])
@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(top_k=40, top_p=0.9), dict(), dict(min_p=0.02, top_p=0.95),
                                dict(temperature=0.0)])
def test_more_rows_than_compute_units(vocab, rows, kw):
    x, u = flat_rows(rows, rows, vocab, torch.float32, 1.0)
    x[::2] *= 2.0  # every other row peaked
    check(x, u, **kw)


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steep", [1.15, 1.3, 1.45])
def test_nuclei_of_hundreds(steep, dtype, rows):
    """More than a wave ranks, and few ids that hold much of what the nucleus leaves."""
    check(*flat_rows(int(100 * steep), rows, 16411, dtype, steep), top_p=0.9)


def test_wide_nuclei_that_no_sample_shows():
    """Rows of one value; of two; weights that only a stretch of ids has; ids in falling and rising order."""
    v = 49152
    x = torch.zeros(6, v)
    x[1, ::3] = -0.01
    x[2] = -30.0
    x[2, 7000:7400] = torch.randn(400, generator=torch.Generator().manual_seed(1))
    x[3] = -torch.arange(v) * (8.0 / v)
    x[4] = torch.arange(v) * (8.0 / v)
    x[5, : v // 2] = -20.0
    for top_p in (0.9, 0.5, 0.999):
        check(x, torch.tensor([0.3, 0.7, 0.5, 0.99, 0.01, 0.6]), top_p=top_p)


@pytest.mark.parametrize("min_p", [0.0, 1e-30, 0.01, 0.1, 0.5, 1.0])
def test_min_p(min_p):
    check(*rows_of(8, 3, 9001), min_p=min_p, temperature=1.3)


@pytest.mark.parametrize("temperature", [0.0, 1e-3, 0.2, 1.0, 10.0, 1e4])
def test_temperatures(temperature):
    check(*rows_of(9, 4, 5003), temperature=temperature)


@pytest.mark.parametrize("seed", range(6))
def test_together(seed):
    g = torch.Generator().manual_seed(seed)
    rows, vocab = 12, [313, 4096, 49152][seed % 3]
    x, u = rows_of(seed, rows, vocab, [torch.float32, torch.bfloat16][seed % 2], [1.0, 4.0][seed // 3])
    pick = lambda values, dt: torch.tensor(values, dtype=dt)[torch.randint(0, len(values), (rows,), generator=g)]
    check(x, u, pick([0.0, 0.5, 0.8, 1.0, 2.0], torch.float32), pick([0, 1, 3, 40, 300], torch.int32),
          pick([1.0, 0.9, 0.5, 0.99], torch.float32), pick([0.0, 0.02, 0.3], torch.float32))


@pytest.mark.parametrize("top_k", [0, 1, 3, 64, 1000, 2000])
@pytest.mark.parametrize("top_p", [1.0, 0.5, 0.25])
def test_ties_go_to_the_lower_id(top_k, top_p):
    """Rows of one value, and of two: borders fall inside the ties."""
    x = torch.zeros(3, 2048)
    x[1, ::2] = -1.0
    x[2] = torch.where(torch.arange(2048) % 3 == 1, 0.0, -0.0)
    check(x, torch.tensor([0.999, 0.3, 0.0]), top_k=top_k, top_p=top_p)


def test_uniforms_at_their_ends():
    x, _ = rows_of(10, 6, 3001)
    x[:, 0] = -50.0
    x[:, -1] = -200.0
    u = torch.tensor([0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0])
    check(x, u)
    check(x, u, top_k=10)
    odd = torch.tensor([-1.0, float("nan"), 1.0, 2.0, float("inf"), -float("inf")])
    got = ops.sample(x.cuda(), odd.cuda(), top_k=10).cpu().tolist()
    first, last = (sorted(torch.topk(x[r], 10).indices.tolist()) for r in (0, 2))
    assert got[0] == first[0] and got[2] == last[-1]
    assert all(0 <= t < 3001 for t in got)


def test_infinities_and_nan():
    inf, nan = float("inf"), float("nan")
    x, u = rows_of(11, 9, 700)
    x[0] = -inf                       # no candidate
    x[1] = nan
    x[2, ::2] = nan
    x[3, 5:] = -inf
    x[4] = -inf
    x[4, 699] = -3e38                 # one candidate, the last
    x[5, 10] = x[5, 600] = inf        # two that share everything
    x[6] = torch.finfo(torch.float32).min
    x[7, 3] = torch.finfo(torch.float32).max
    x[8] = torch.finfo(torch.float32).min
    x[8, 9:] = -inf
    for kw in ({}, {"top_k": 3}, {"top_p": 0.6}, {"min_p": 0.2}, {"temperature": 0.0}, {"top_k": 650, "top_p": 0.99}):
        got = check(x, u, **kw)
        assert got[0] == -1 and got[1] == -1 and got[4] == 699 and got[5] in (10, 600)


def test_strides_and_shapes():
    x, u = rows_of(12, 12, 333)
    want = ops.sample(x.cuda(), u.cuda(), 0.9, 20)
    wide = torch.zeros(12, 400, device="cuda")
    wide[:, 3:336] = x.cuda()
    assert torch.equal(ops.sample(wide[:, 3:336], u.cuda(), 0.9, 20), want)
    assert torch.equal(ops.sample(x.t().contiguous().cuda().t(), u.cuda(), 0.9, 20), want)
    got = ops.sample(x.view(3, 4, 333).cuda(), u.view(3, 4).cuda(), 0.9, 20)
    assert got.shape == (3, 4) and torch.equal(got.view(-1), want)
    assert ops.sample(x[0].cuda(), u[0].cuda(), 0.9, 20).shape == ()
    assert torch.equal(ops.sample(x[:1].expand(12, 333).cuda(), u.cuda(), 0.9, 20)[0], want[0])
    out = torch.zeros(12, dtype=torch.int64, device="cuda")
    probs = torch.full((12, 340), 5.0, device="cuda")
    assert ops.sample(x.cuda(), u.cuda(), 0.9, 20, out=out, probs=probs[:, 2:335]) is out and torch.equal(out, want)
    assert bool((probs[:, :2] == 5).all()) and bool((probs[:, 335:] == 5).all())
    assert ops.sample(x[:0].cuda(), u[:0].cuda()).shape == (0,)


def test_frequencies_follow_the_distribution():
    """20000 even uniforms: each kept id gets its share to within one of them."""
    x, _ = rows_of(13, 1, 501)
    n = 20000
    u = (torch.arange(n) + 0.5) / n
    got = ops.sample(x.expand(n, 501).cuda(), u.cuda(), 0.9, top_k=30, top_p=0.95).cpu()
    _, p, _ = draw(x[0], 0.5, float(torch.tensor(0.9)), 30, float(torch.tensor(0.95)), 0.0)
    share = torch.bincount(got, minlength=501).double()
    assert bool(((share - n * p).abs() <= 1.0 + n * 2.0 ** -24 * 4).all())


def test_captured_and_replayed():
    x, u = rows_of(14, 5, 30001)
    y, w = rows_of(15, 5, 30001)
    xs, us = x.cuda(), u.cuda()
    run = lambda: ops.sample(xs, us, 0.8, 40, 0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for a, b in ((y, w), (x, u), (y, w)):
        xs.copy_(a)
        us.copy_(b)
        want = run().clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_wrapper_refuses():
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    row = torch.zeros(3, device="cuda")
    wrong = [
        (TypeError, dict(logits=x.half())), (ValueError, dict(logits=x[:, :0])), (ValueError, dict(u=u[:2])),
        (TypeError, dict(u=u.double())), (RuntimeError, dict(u=u.cpu())), (ValueError, dict(temperature=-0.1)),
        (ValueError, dict(temperature=float("nan"))), (ValueError, dict(temperature=float("inf"))),
        (ValueError, dict(top_k=-1)), (ValueError, dict(top_p=1.1)), (ValueError, dict(top_p=-0.1)),
        (ValueError, dict(min_p=2.0)), (TypeError, dict(temperature=row.double())), (ValueError, dict(top_p=row[:2])),
        (TypeError, dict(top_k=row)), (TypeError, dict(out=row)), (ValueError, dict(out=torch.zeros(2, dtype=torch.int64, device="cuda"))),
        (ValueError, dict(probs=torch.zeros(3, 9, device="cuda"))), (TypeError, dict(probs=x.double())),
        (ValueError, dict(probs=x[:1].expand(3, 10))), (ValueError, dict(probs=torch.zeros(10, 3, device="cuda").t())),
    ]
    for kind, change in wrong:
        with pytest.raises(kind):
            ops.sample(**{**dict(logits=x, u=u), **change})
