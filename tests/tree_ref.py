"""Trees of drafted tokens, paged caches and the operators' definitions in 64
bits on the CPU, for the tests of the tree operators."""
import numpy as np
import torch


def random_parents(rng, batch, nodes, reach=None):
    """parents [batch, nodes], -1 at node 0, each node's among the `reach` before it (all where None)."""
    parents = np.full((batch, nodes), -1, dtype=np.int32)
    for i in range(1, nodes):
        parents[:, i] = rng.integers(0 if reach is None else max(0, i - reach), i, batch)
    return torch.from_numpy(parents)


def ancestors(parents):
    """(seen bool [B, N, N], itself among them, depth int32 [B, N])"""
    b, n = parents.shape
    seen = torch.zeros(b, n, n, dtype=torch.bool)
    depth = torch.zeros(b, n, dtype=torch.int32)
    for r in range(b):
        for i in range(n):
            seen[r, i, i] = True
            p = int(parents[r, i])
            if p >= 0:
                seen[r, i] |= seen[r, p]
                depth[r, i] = depth[r, p] + 1
    return seen, depth


def words(seen):
    """seen [B, Q, N] as bits of int64 [B, Q, ceil(N / 64)]"""
    b, q, n = seen.shape
    padded = np.zeros((b, q, -(-n // 64) * 64), dtype=np.uint8)
    padded[:, :, :n] = seen.numpy()
    return torch.from_numpy(np.packbits(padded, axis=2, bitorder="little").view(np.int64).copy())


def rope_tables(positions, dim, theta=10000.0):
    inv = 1.0 / theta ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim)
    angle = torch.arange(positions, dtype=torch.float32)[:, None] * inv
    return angle.cos(), angle.sin()


def rotate(x, cos, sin):
    """x [..., heads, dim] rotated in fp32, product by product, and rounded to its type."""
    x1, x2 = x.float().chunk(2, -1)
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).to(x.dtype)


class Case:
    """Inputs of one tree_attention call on the CPU."""

    def __init__(self, seed, past, nodes, heads, kv, dim=64, bs=16, dtype=torch.bfloat16, first=0, live=None,
                 parents=None, seen=None, spare=0):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        batch = len(past)
        self.past, self.nodes, self.heads, self.kv, self.dim, self.bs, self.first = past, nodes, heads, kv, dim, bs, first
        self.live = [nodes] * batch if live is None else live
        self.parents = random_parents(rng, batch, nodes) if parents is None else parents
        got, self.depth = ancestors(self.parents)
        self.seen = got if seen is None else seen
        self.mask = words(self.seen[:, first:])
        cols = [-(-(p + spare) // bs) for p in past]
        blocks = sum(cols) + 2
        ids = torch.from_numpy(rng.permutation(blocks).astype(np.int32))
        self.tables = torch.full((batch + 1, max(cols) + 1), blocks - 1, dtype=torch.int32)
        # the rows of the tables in another order than the batch's
        self.rows = rng.permutation(batch + 1)[:batch]
        at = 0
        for b in range(batch):
            self.tables[self.rows[b], :cols[b]] = ids[at:at + cols[b]]
            at += cols[b]
        self.k_pool = torch.randn(blocks, kv, bs, dim, generator=g).to(dtype)
        self.v_pool = torch.randn(blocks, kv, dim, bs, generator=g).to(dtype)
        self.qkv = torch.randn(batch, nodes, (heads + 2 * kv) * dim, generator=g).to(dtype)
        self.qkv[:, :, :heads * dim] *= 1.5
        self.cos, self.sin = rope_tables(max(past) + nodes + 1, dim)
        self.meta = torch.tensor([list(map(int, self.rows)), past, self.live], dtype=torch.int32)
        self.scale = dim ** -0.5

    def call(self, ops, dev="cuda", **kw):
        t = {n: getattr(self, n).to(dev) for n in ("qkv", "cos", "sin", "k_pool", "v_pool", "tables", "meta", "mask",
                                                   "depth")}
        t.update(n_heads=self.heads, scale=self.scale, max_kv_len=max(self.past), first=self.first)
        t.update(kw)
        return ops.tree_attention(**t)

    def reference(self):
        """(out, spread) float64 [B, N - first, H * dim]: the attention and sum
        p |v| / sum p, and the largest sum |q k| * scale of the call; NaN where
        a query is not live."""
        batch, width = len(self.past), self.nodes - self.first
        out = torch.full((batch, width, self.heads, self.dim), float("nan"), dtype=torch.float64)
        spread = out.clone()
        reach = 0.0
        for b in range(batch):
            live, past = min(self.live[b], self.nodes), self.past[b]
            if live <= self.first:
                continue
            x = self.qkv[b, :live].view(live, -1, self.dim)
            at = past + self.depth[b, :live].long()
            c, s = self.cos[at][:, None], self.sin[at][:, None]
            q = rotate(x[:, :self.heads], c, s)[self.first:].double()
            k = rotate(x[:, self.heads:self.heads + self.kv], c, s).double()
            ids = self.tables[self.rows[b], :-(-past // self.bs)].long()
            for h in range(self.heads):
                hk = h // (self.heads // self.kv)
                keys = torch.cat([self.k_pool[ids, hk].reshape(-1, self.dim)[:past].double(), k[:, hk]])
                vals = torch.cat([self.v_pool[ids, hk].transpose(1, 2).reshape(-1, self.dim)[:past].double(),
                                  x[:, self.heads + self.kv + hk].double()])
                z = q[:, h] @ keys.t() * self.scale
                see = torch.cat([torch.ones(live - self.first, past, dtype=torch.bool),
                                 self.seen[b, self.first:live, :live]], 1)
                reach = max(reach, float((q[:, h].abs() @ keys.abs().t()).max()) * self.scale)
                z = z.masked_fill(~see, float("-inf"))
                p = torch.where(see, torch.exp(z - z.amax(1, keepdim=True)), torch.zeros_like(z))
                p = torch.where(see.any(1, keepdim=True), p / p.sum(1, keepdim=True), torch.zeros_like(p))
                out[b, :live - self.first, h] = p @ vals
                spread[b, :live - self.first, h] = p @ vals.abs()
        return out.flatten(2), spread.flatten(2), reach

    def tolerance(self, out, spread, reach):
        """|kernel - reference| at most, from the roundings that the kernel makes.

        Scores: dim products added in fp32, each step at most 2^-24 of sum
        |q k|, and the scaling's; a score off by e moves each weight by e
        relative, so the output by 2 e spread.  Weights: exp within 4 steps of
        2^-24 and, in bf16, rounded for the product (2^-8).  Sums over n keys
        in fp32: n 2^-24 of the spread at worst, numerator and denominator.
        Output: one rounding."""
        half = torch.finfo(self.qkv.dtype).eps / 2
        n = max(self.past) + self.nodes
        e = (self.dim + 4) * 2.0 ** -24 * reach
        weight = 4 * 2.0 ** -24 + (half if self.qkv.dtype == torch.bfloat16 else 0.0)
        off = (2 * e + weight + 2 * (n + 8) * 2.0 ** -24) * spread
        return off + half * (out.abs() + off) + 1e-30


def walk(tokens, parents, sampled, live, room):
    """The accepted path of one row, node 0 first ([] for a row of none)."""
    live = min(live, len(tokens))
    if live <= 0:
        return []
    way = [0]
    while len(way) < room:
        child = [c for c in range(way[-1] + 1, live)
                 if int(parents[c]) == way[-1] and int(tokens[c]) == int(sampled[way[-1]])]
        if not child:
            break
        way.append(child[0])
    return way


def draw(x, u, temperature, top_k, top_p, min_p):
    """(token, probabilities float64 [V]) of one row of logits by sorting, in 64
    bits; also the distance of u from the nearest border of its token, relative
    to the total."""
    x = torch.where(x.isnan(), torch.full_like(x, float("-inf")), x).double()
    v = len(x)
    none = torch.zeros(v, dtype=torch.float64)
    if bool((x == float("-inf")).all()):
        return -1, none, 1.0
    ids = torch.argsort(x, descending=True, stable=True)
    if not temperature > 0:
        ids = ids[:1]
    elif top_k > 0:
        ids = ids[:top_k]
    top = x[ids[0]]
    w = torch.where(x[ids] == top, torch.ones(len(ids), dtype=torch.float64),
                    torch.exp((x[ids] - top) / (temperature if temperature > 0 else 1.0)))
    mass = w.cumsum(0)
    keep = len(ids)
    if temperature > 0:
        if top_p < 1:
            keep = min(keep, max(1, int((torch.cat([none[:1], mass[:-1]]) < top_p * mass[-1]).sum())))
        if min_p > 0:
            keep = min(keep, max(1, int((w >= min_p).sum())))
    row = none.clone()
    row[ids[:keep]] = w[:keep]
    run = row.cumsum(0)
    want = u * run[-1]
    over = ((run > want) & (row > 0)).nonzero()
    token = int(over[0]) if len(over) else int((row > 0).nonzero()[-1])
    gap = float((run - want).abs().min() / run[-1])
    return token, row / run[-1], gap
