"""Tree attention and the commit of an accepted path against their definitions
in 64 bits."""
import numpy as np
import pytest
import torch

from specdec import ops
from tree_ref import Case, random_parents, rope_tables, rotate, walk

pytestmark = pytest.mark.gpu


def check(case, **kw):
    out, spread, reach = case.reference()
    batch, width = len(case.past), case.nodes - case.first
    into = torch.full((batch, width, case.heads * case.dim), 7.0, dtype=case.qkv.dtype, device="cuda")
    got = case.call(ops, out=into, **kw)
    assert got is into
    got = got.cpu().double()
    live = ~out.isnan()
    off = (got - out).abs()[live]
    tol = case.tolerance(out, spread, reach)[live]
    assert bool((off <= tol).all()), (float((off / tol).max()), float(off.max()))
    assert bool((got[~live] == 7.0).all())  # queries that are not live stay as they were
    return got


HEADS = [(4, 4), (9, 3), (8, 2), (8, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv", HEADS)
@pytest.mark.parametrize("dim", [64, 128])
def test_heads_and_types(dtype, heads, kv, dim):
    check(Case(heads * dim, [70, 3], 12, heads, kv, dim, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("past", [0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 130, 255, 257, 511, 513, 1000, 2049])
def test_cached_lengths(dtype, past):
    check(Case(past, [past], 7, 4, 2, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes", [1, 2, 5, 15, 16, 17, 31, 33, 63, 64, 65, 100, 128, 129, 200, 256])
def test_tree_sizes(dtype, nodes):
    check(Case(nodes, [37, 90], nodes, 4, 2, dtype=dtype))


@pytest.mark.parametrize("bs", [1, 3, 8, 12, 16, 24, 32, 40, 64, 100, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_sizes(bs, dtype):
    check(Case(bs, [99, 300], 9, 6, 3, bs=bs, dtype=dtype))


@pytest.mark.parametrize("first", [1, 4, 13, 20, 21])
@pytest.mark.parametrize("nodes", [21, 80])
def test_later_levels_alone(first, nodes):
    """The nodes from `first` on give the rows that the whole tree's call gives them."""
    case = Case(first, [50, 200, 1], nodes, 9, 3, first=first)
    check(case)


@pytest.mark.parametrize("heads,kv,nodes", [(32, 32, 16), (32, 8, 64), (16, 1, 40), (9, 3, 33)])
def test_many_query_rows(heads, kv, nodes):
    check(Case(nodes, [200, 77], nodes, heads, kv))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv,nodes,first", [(4, 2, 24, 0), (8, 2, 40, 0), (8, 1, 65, 3), (2, 2, 100, 40)])
@pytest.mark.parametrize("past", [[63, 64], [2000, 1], [4097, 900]])
def test_many_query_rows_at_any_length(dtype, dim, heads, kv, nodes, first, past):
    """48 to 496 query rows a kv head, splits of one and several chunks, ends inside chunks and pages."""
    check(Case(nodes + past[0], past, nodes, heads, kv, dim, dtype=dtype, first=first, bs=16 if dim == 64 else 24))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes", [12, 50, 90])
def test_values_that_are_no_numbers_reach_who_sees_them(dtype, nodes):
    """An infinite value of a node makes the outputs of the queries that see it
    infinite, and no others'."""
    case = Case(30, [40, 700], nodes, 8, 2, dtype=dtype)
    want, spread, reach = case.reference()
    at = (8 + 2) * 64 + 5  # v of kv head 0, dim 5
    case.qkv[0, 3, at] = float("inf")
    case.qkv[0, 3, at + 64] = float("nan")  # kv head 1
    got = case.call(ops).cpu().double().view(2, nodes, 8, 64)
    sees = case.seen[0, :, 3]
    assert bool((got[0, sees, :4, 5] == float("inf")).all()) and bool(got[0, sees, 4:, 5].isnan().all())
    ok = torch.ones(2, nodes, 8, 64, dtype=torch.bool)
    ok[0, sees, :, 5] = False
    off = (got - want.view_as(got)).abs()
    assert bool((off <= case.tolerance(want, spread, reach).view_as(got))[ok].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_different_sizes(dtype):
    """Ragged lengths, rows of few live nodes and of none."""
    check(Case(5, [0, 1, 700, 64, 33, 128], 20, 4, 4, live=[20, 1, 7, 0, 19, 20], dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_that_leave_nothing(dtype):
    """A query that sees neither cache nor node gets zeros; any mask is taken, its
    own bit not implied."""
    nodes = 70
    rng = np.random.default_rng(3)
    seen = torch.from_numpy(rng.random((3, nodes, nodes)) < 0.2)
    seen[:, 0] = False
    seen[0, 5] = False
    seen[1, 65:] = False
    got = check(Case(6, [0, 0, 40], nodes, 4, 2, seen=seen, dtype=dtype))
    assert bool((got[0, 5] == 0).all()) and bool((got[1, 69] == 0).all())


@pytest.mark.parametrize("more", [0, 40])
def test_nan_and_infinity_where_nothing_looks(more):
    """Values behind the cached length, of nodes that are not live or not seen, and of other rows' blocks."""
    case = Case(8, [37, 20], 12 + more, 4, 2, live=[12 + more, 9])
    seen_by_none = 7
    case.seen[0, :, seen_by_none] = False
    case.seen[0, seen_by_none, seen_by_none] = False
    from tree_ref import words
    case.mask = words(case.seen)
    want, spread, reach = case.reference()
    for b in range(2):
        last = case.tables[case.rows[b], case.past[b] // 16]
        case.k_pool[last, :, case.past[b] % 16:] = float("nan")
        case.v_pool[last, :, :, case.past[b] % 16:] = float("inf")
    used = set(case.tables[case.rows[0], :3].tolist()) | set(case.tables[case.rows[1], :2].tolist())
    for i in range(case.k_pool.shape[0]):
        if i not in used:
            case.k_pool[i], case.v_pool[i] = float("nan"), float("nan")
    case.qkv[1, 9:] = float("nan")
    q_end = 4 * 64
    case.qkv[0, seen_by_none, q_end:q_end + 128] = float("inf")
    case.qkv[0, seen_by_none, q_end + 128:] = float("nan")
    got = case.call(ops).cpu().double()
    live = ~want.isnan()
    assert bool(((got - want).abs() <= case.tolerance(want, spread, reach))[live].all())


def test_nan_in_a_seen_place_reaches_the_rows_that_see_it_alone():
    case = Case(9, [20, 20], 6, 2, 2)
    case.qkv[0, 3, 2 * 64:3 * 64] = float("nan")  # node 3's key of head 0
    got = case.call(ops).cpu().view(2, 6, 2, 64)
    assert bool(got[0, case.seen[0, :, 3], 0].isnan().all())
    assert not bool(got[0, ~case.seen[0, :, 3], 0].isnan().any())
    assert not bool(got[0, :, 1].isnan().any()) and not bool(got[1].isnan().any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes", [12, 90])
def test_strided_operands_and_shared_trees(dtype, nodes):
    """qkv and out as parts of wider buffers, the mask and depths of one tree for every row."""
    rng = np.random.default_rng(4)
    parents = random_parents(rng, 1, nodes).expand(3, nodes).contiguous()
    case = Case(10, [33, 90, 5], nodes, 4, 2, dtype=dtype, parents=parents)
    want = check(case)
    wide = torch.zeros(3, nodes + 2, case.qkv.shape[2] + 40, dtype=dtype, device="cuda")
    wide[:, 1:-1, 8:-32] = case.qkv.cuda()
    out = torch.full((3, nodes + 1, 4 * 64 + 24), 3.0, dtype=dtype, device="cuda")
    got = case.call(ops, qkv=wide[:, 1:-1, 8:-32], out=out[:, 1:, 16:-8], mask=case.mask[:1].cuda(),
                    depth=case.depth[:1].cuda())
    assert torch.equal(got.cpu().double(), want)
    assert bool((out[:, 0] == 3).all()) and bool((out[:, :, :16] == 3).all()) and bool((out[:, :, -8:] == 3).all())
    # rows whose addresses allow no wide loads
    odd = torch.zeros(3, nodes, case.qkv.shape[2] + 3, dtype=dtype, device="cuda")
    odd[:, :, 1:-2] = case.qkv.cuda()
    off = (case.call(ops, qkv=odd[:, :, 1:-2]).cpu().double() - want).abs()
    ref, spread, reach = case.reference()
    assert bool((off <= 2 * case.tolerance(ref, spread, reach)).all())


def test_mask_of_whole_rows_and_two_dimensions():
    case = Case(11, [33, 9], 10, 4, 2)
    assert torch.equal(case.call(ops), case.call(ops, mask=case.mask[:, :, 0].cuda()))


def test_max_kv_len_is_a_layout_only():
    """Rows longer than max_kv_len, and much shorter, are right."""
    case = Case(12, [900, 20], 9, 4, 2)
    for most in (0, 1, 64, 300, 5000, 100000):
        check(case, max_kv_len=most)


@pytest.mark.parametrize("nodes,bs", [(5, 16), (5, 10), (60, 16)])
def test_bad_metadata_reads_nothing_out_of_range(nodes, bs):
    """A table row, past or block id outside the tables and the pool, a position
    outside the rotation's tables: NaN in the rows concerned, the others right."""
    case = Case(13, [40, 40, 40, 40, 40, 40, 40], nodes, 4, 2, bs=bs)
    want = case.call(ops).cpu()
    meta, tables, depth = case.meta.clone(), case.tables.clone(), case.depth.clone()
    meta[0, 0] = 1000
    meta[0, 1] = -1
    meta[1, 2] = -5
    meta[1, 3] = 1 << 30
    tables[case.rows[4], 1] = case.k_pool.shape[0]
    tables[case.rows[5], 2] = -7
    depth[6, 4] = 1 << 30
    got = case.call(ops, meta=meta.cuda(), tables=tables.cuda(), depth=depth.cuda()).cpu()
    assert bool(got[:6].isnan().all())
    blind = ~case.seen[6, :, 4]
    assert torch.equal(got[6, blind], want[6, blind]) and bool(got[6, ~blind].isnan().all())


def test_large_offsets():
    """A pool past 2^32 bytes, its last blocks in use."""
    case = Case(14, [50, 33], 9, 8, 8)
    blocks = case.k_pool.shape[0]
    total = (1 << 32) // (8 * 16 * 64 * 2) + 64
    k = torch.full((total, 8, 16, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    v = torch.full((total, 8, 64, 16), float("nan"), dtype=torch.bfloat16, device="cuda")
    k[total - blocks:] = case.k_pool.cuda()
    v[total - blocks:] = case.v_pool.cuda()
    tables = (case.tables + (total - blocks)).cuda()
    assert torch.equal(case.call(ops), case.call(ops, k_pool=k, v_pool=v, tables=tables))


def test_runs_are_the_same_bits_and_streams_do_not_meet():
    case = Case(15, [3000 - 7, 1200], 24, 4, 4)
    want = case.call(ops)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(case.call(ops))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_captured_and_replayed():
    """A captured call follows its inputs, lengths and table among them."""
    a, b = Case(16, [300, 20], 10, 4, 2, spare=0), Case(17, [100, 290], 10, 4, 2)
    names = ("qkv", "k_pool", "v_pool", "tables", "meta", "mask", "depth")
    blocks = max(a.k_pool.shape[0], b.k_pool.shape[0])
    cols = max(a.tables.shape[1], b.tables.shape[1])

    def widened(c):
        t = {n: getattr(c, n) for n in names}
        t["k_pool"] = torch.cat([c.k_pool, torch.zeros(blocks - c.k_pool.shape[0], *c.k_pool.shape[1:], dtype=c.k_pool.dtype)])
        t["v_pool"] = torch.cat([c.v_pool, torch.zeros(blocks - c.v_pool.shape[0], *c.v_pool.shape[1:], dtype=c.v_pool.dtype)])
        t["tables"] = torch.nn.functional.pad(c.tables, (0, cols - c.tables.shape[1]))
        return {n: x.cuda() for n, x in t.items()}

    held, other = widened(a), widened(b)
    cos, sin = (t.cuda() for t in rope_tables(400, 64))
    run = lambda: ops.tree_attention(held["qkv"], cos, sin, held["k_pool"], held["v_pool"], held["tables"], held["meta"],
                                     held["mask"], held["depth"], 4, 0.125, 512)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    first = {n: held[n].clone() for n in names}
    for source in (first, other, first, other):
        for n in names:
            held[n].copy_(source[n])
        want = run().clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ------------------------------------------------------------------- commit --
class Commit:
    def __init__(self, seed, past, nodes, layers=3, heads=4, kv=2, dim=64, bs=16, dtype=torch.bfloat16, room=None,
                 live=None, vocab=5):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        batch = len(past)
        self.past, self.nodes, self.heads, self.kv, self.dim, self.bs, self.layers = past, nodes, heads, kv, dim, bs, layers
        self.room = nodes if room is None else room
        self.live = [nodes] * batch if live is None else live
        self.parents = random_parents(rng, batch, nodes, reach=4)
        self.tokens = torch.randint(0, vocab, (batch, nodes), generator=g)
        self.sampled = torch.randint(0, vocab, (batch, nodes), generator=g)
        cols = max(-(-(p + self.room) // bs) for p in past)
        blocks = batch * cols + 3
        self.tables = torch.from_numpy(rng.permutation(blocks)[:batch * cols].reshape(batch, cols).astype(np.int32))
        self.k_pool = torch.randn(layers, blocks, kv, bs, dim, generator=g).to(dtype)
        self.v_pool = torch.randn(layers, blocks, kv, dim, bs, generator=g).to(dtype)
        self.qkv = torch.randn(layers, batch, nodes, (heads + 2 * kv) * dim, generator=g).to(dtype)
        self.cos, self.sin = rope_tables(max(past) + nodes + 1, dim)
        self.meta = torch.tensor([list(range(batch)), past, self.live], dtype=torch.int32)

    def want(self):
        k_pool, v_pool = self.k_pool.clone(), self.v_pool.clone()
        batch = len(self.past)
        verdict = torch.full((self.nodes + 1, batch), -1, dtype=torch.int64)
        path = torch.full((batch, self.nodes), -1, dtype=torch.int32)
        for b in range(batch):
            way = walk(self.tokens[b], self.parents[b], self.sampled[b], self.live[b], self.room)
            verdict[0, b] = len(way) - 1
            if way:
                verdict[1, b] = self.sampled[b, way[-1]]
            for j, c in enumerate(way):
                path[b, j] = c
                if j:
                    verdict[1 + j, b] = self.tokens[b, c]
                at = self.past[b] + j
                block, slot = int(self.tables[b, at // self.bs]), at % self.bs
                x = self.qkv[:, b, c].view(self.layers, -1, self.dim)
                k_pool[:, block, :, slot] = rotate(x[:, self.heads:self.heads + self.kv], self.cos[at], self.sin[at])
                v_pool[:, block, :, :, slot] = x[:, self.heads + self.kv:]
        return verdict, path, k_pool, v_pool

    def call(self, **kw):
        t = {n: getattr(self, n).cuda() for n in ("tokens", "parents", "sampled", "meta", "qkv", "cos", "sin", "k_pool",
                                                  "v_pool", "tables")}
        t.update(room=self.room)
        t.update(kw)
        return (*ops.tree_commit(**t), t["k_pool"], t["v_pool"])

    def check(self, **kw):
        for name, got, want in zip(("verdict", "path", "k", "v"), self.call(**kw), self.want()):
            assert torch.equal(got.cpu(), want), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes", [1, 2, 7, 16, 63, 64, 65, 130, 256])
def test_commit_of_random_trees(dtype, nodes):
    """Few tokens, so paths go deep and siblings carry the same one."""
    Commit(nodes, [0, 5, 15, 16, 40, 100], nodes, vocab=3, dtype=dtype).check()


@pytest.mark.parametrize("dim,heads,kv", [(64, 9, 3), (128, 8, 1), (32, 4, 4), (2, 1, 1), (80, 3, 1)])
@pytest.mark.parametrize("bs", [1, 5, 16, 64])
def test_commit_heads_and_blocks(dim, heads, kv, bs):
    Commit(dim + bs, [3, 30], 20, heads=heads, kv=kv, dim=dim, bs=bs, vocab=2).check()


@pytest.mark.parametrize("room", [1, 2, 4, 100])
def test_commit_stops_at_its_room(room):
    case = Commit(room, [3, 30, 7], 40, room=room, vocab=1)
    case.check()
    assert int(case.want()[0][0].max()) == min(room - 1, int(case.want()[0][0].max()))


def test_commit_of_rows_with_few_live_nodes():
    Commit(2, [3, 30, 7, 9], 30, live=[0, 1, 5, 30], vocab=2).check()


def test_commit_of_one_tree_for_every_row():
    case = Commit(3, [3, 30, 7], 30, vocab=2)
    case.parents = case.parents[:1].expand(3, 30)
    case.check(parents=case.parents[:1].contiguous().cuda())


def test_walk_alone():
    case = Commit(4, [3, 30, 7], 30, vocab=2)
    verdict, path = ops.tree_commit(case.tokens.cuda(), case.parents.cuda(), case.sampled.cuda(), case.meta.cuda())
    want = case.want()
    assert torch.equal(verdict.cpu(), want[0]) and torch.equal(path.cpu(), want[1])


def test_commit_ends_before_a_slot_that_is_none():
    """A table row, a block id or a position outside: the path ends there and nothing else is written."""
    case = Commit(5, [14, 14, 14, 14, 14], 30, vocab=1)
    tables, meta = case.tables.clone(), case.meta.clone()
    tables[1, 1] = -1                       # the second block: two slots are left
    tables[2, 1] = case.k_pool.shape[1]
    meta[0, 3] = 77
    meta[1, 4] = -3
    verdict, path, k, v = case.call(tables=tables.cuda(), meta=meta.cuda())
    whole = case.want()
    case.tables, case.room = case.tables, 2
    short = case.want()
    assert torch.equal(verdict[:, 0].cpu(), whole[0][:, 0])
    assert torch.equal(verdict[:, 1:3].cpu(), short[0][:, 1:3]) and torch.equal(path[1:3].cpu(), short[1][1:3])
    assert verdict[:, 3:].cpu().tolist() == [[-1, -1]] * 31
    want_k, want_v = case.k_pool.clone(), case.v_pool.clone()
    for b, pool in ((0, whole), (1, short), (2, short)):
        ids = case.tables[b].long()
        want_k[:, ids], want_v[:, ids] = pool[2][:, ids], pool[3][:, ids]
    assert torch.equal(k.cpu(), want_k) and torch.equal(v.cpu(), want_v)


def test_commit_of_strided_projections_twice():
    """qkv as part of a wider buffer; a second call gives the same."""
    case = Commit(6, [3, 30], 12, vocab=2)
    wide = torch.zeros(3, 2, 15, case.qkv.shape[3] + 9, dtype=case.qkv.dtype, device="cuda")
    view = wide[:, :, 2:14, 5:-4]
    view.copy_(case.qkv)
    k, v = case.k_pool.cuda(), case.v_pool.cuda()
    for _ in range(2):
        case.check(qkv=view, k_pool=k, v_pool=v)


# ----------------------------------------------------------------- refusals --
def test_attention_wrapper_refuses():
    """Each refusal comes before a launch."""
    case = Case(20, [30, 9], 10, 4, 2)
    gpu = {n: getattr(case, n).cuda() for n in ("qkv", "cos", "sin", "k_pool", "v_pool", "tables", "meta", "mask", "depth")}
    good = lambda: torch.empty(2, 10, 256, dtype=torch.bfloat16, device="cuda")
    wrong = [
        (TypeError, dict(qkv=gpu["qkv"].half())), (ValueError, dict(qkv=gpu["qkv"][0])),
        (TypeError, dict(k_pool=gpu["k_pool"].float())), (ValueError, dict(k_pool=gpu["k_pool"][0])),
        (ValueError, dict(v_pool=gpu["k_pool"])), (ValueError, dict(k_pool=gpu["k_pool"][:, :, ::2])),
        (ValueError, dict(qkv=gpu["qkv"][:, :, :-64])), (ValueError, dict(n_heads=2)), (ValueError, dict(first=11)),
        (ValueError, dict(first=-1)), (ValueError, dict(cos=gpu["cos"][:, :16])), (TypeError, dict(sin=gpu["sin"].double())),
        (TypeError, dict(tables=gpu["tables"].long())), (ValueError, dict(tables=gpu["tables"].t())),
        (TypeError, dict(meta=gpu["meta"].long())), (ValueError, dict(meta=gpu["meta"][:2])),
        (ValueError, dict(mask=gpu["mask"][:, :9])), (TypeError, dict(mask=gpu["mask"].int())),
        (ValueError, dict(first=2)), (ValueError, dict(depth=gpu["depth"][:, :9])), (TypeError, dict(depth=gpu["depth"].long())),
        (ValueError, dict(out=good()[:, :9])), (TypeError, dict(out=good().float())), (RuntimeError, dict(out=good().cpu())),
        (ValueError, dict(out=good()[:, :1].expand(2, 10, 256))), (RuntimeError, dict(mask=case.mask)),
        (RuntimeError, dict(max_kv_len=-1)),
    ]
    for kind, change in wrong:
        with pytest.raises(kind):
            case.call(ops, **change)
    odd = Case(21, [30], 5, 2, 2, dim=32)
    with pytest.raises(NotImplementedError):
        odd.call(ops)
    big = torch.zeros(1, 257, 6 * 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        case.call(ops, qkv=big)
    assert case.call(ops, qkv=gpu["qkv"][:0], mask=gpu["mask"][:0], depth=gpu["depth"][:0],
                     meta=gpu["meta"][:, :0].contiguous()).shape == (0, 10, 256)


def test_commit_wrapper_refuses():
    case = Commit(7, [3, 30], 12)
    gpu = {n: getattr(case, n).cuda() for n in ("tokens", "parents", "sampled", "meta", "qkv", "cos", "sin", "k_pool",
                                                "v_pool", "tables")}
    wrong = [
        (TypeError, dict(tokens=gpu["tokens"].int())), (ValueError, dict(tokens=gpu["tokens"][0])),
        (ValueError, dict(sampled=gpu["sampled"][:1])), (ValueError, dict(sampled=gpu["sampled"][:, :11])),
        (TypeError, dict(parents=gpu["parents"].long())), (ValueError, dict(room=0)), (ValueError, dict(meta=gpu["meta"][:2])),
        (ValueError, dict(qkv=gpu["qkv"][0])), (ValueError, dict(qkv=gpu["qkv"][:2])), (TypeError, dict(qkv=gpu["qkv"].half())),
        (ValueError, dict(qkv=None)), (ValueError, dict(cos=None)), (ValueError, dict(v_pool=None)),
        (ValueError, dict(tables=None)), (ValueError, dict(k_pool=gpu["k_pool"][0])), (TypeError, dict(v_pool=gpu["v_pool"].float())),
        (ValueError, dict(cos=gpu["cos"][:, :4])), (TypeError, dict(tables=gpu["tables"].long())),
    ]
    for kind, change in wrong:
        with pytest.raises(kind):
            case.call(**change)
