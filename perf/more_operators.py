"""The operators of a round that verifies a tree of drafted tokens, as cases that can be timed and checked.

A case is one call of one operator, as a round makes it:

  attn    the attention of a tree's nodes over a paged cache and over one another
          (specdec.ops.tree_attention)
  sample  a token for each row of logits, under temperature, top-k, top-p and
          min-p, from given uniforms; with `probs` also the distribution that it
          was drawn from (specdec.ops.sample)
  commit  the walk down the tree along the sampled tokens, and the accepted
          nodes' keys and values of every layer appended to the cache
          (specdec.ops.tree_commit)

A tree has N nodes, parents before children, node 0 the last token of the
context; a node's depth is its distance from node 0 and its mask has a bit for
itself and for each ancestor.

attn: node j of row b stands at position past[b] + depth[j].  Its q and k are
rotated there (x1 cos - x2 sin, x2 cos + x1 sin for the halves of a head) and
rounded to the activations' type, as a cache holds them.  Query i sees the past[b] cached keys
and the nodes j < nodes[b] of its mask; queries past nodes[b] are not written.

sample: ids in the order of falling logits, ties by the lower id, w = exp((x -
max) / T).  Kept is the shortest of three prefixes: the first top_k; those with w
>= min_p; the least prefix whose mass reaches top_p of the mass of the first
top_k.  The token is the least id whose running sum of kept weights, in the
order of ids, exceeds u times their total; at T = 0 the first of the order.  A
NaN weighs nothing.  Parameters are fp32 (top_k int32), one for the call or one a row.

commit: from node 0, the child (the lowest, where two carry one token) that
carries the token sampled at the node, until there is none.

Sizes are the SmolLM2-1.7B target's and the SmolLM2-135M draft's heads and
vocabulary, grouped heads of the usual kinds, and trees of 8 to 64 nodes.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
THETA = 130000.0


def listed():
    return [
        # one request of the target, a small tree, a short context: latency counts
        _attn("attn_b1_n16_c300", 1, 16, 300, 32, 32),
        # eight requests of the target at a long context
        _attn("attn_b8_n32_c4096", 8, 32, 4096, 32, 32),
        # a level of the draft's own tree: its last 8 nodes are new, one tree for the whole batch
        _attn("attn_b16_n21_c1000_level", 16, 21, 1000, 9, 3, first=13, shared=True),
        # a model in fp32, an odd number of nodes
        _attn("attn_b4_n13_c1500_f32", 4, 13, 1500, 32, 32, dtype="f32"),
        # grouped heads of 128, a wide tree: 256 query rows for each kv head
        _attn("attn_b4_n64_c8000_gqa128", 4, 64, 8000, 32, 8, dim=128, bs=32),
        # the first token after a prompt, one request: nothing cut off
        _sample("sample_1x49152", 1, 49152, temperature=0.8),
        # eight trees of 8 nodes, one setting for the call
        _sample("sample_64x49152_k50_p95", 64, 49152, temperature=0.7, top_k=50, top_p=0.95),
        # 32 trees of 16 nodes, nucleus alone
        _sample("sample_512x49152_p90", 512, 49152, temperature=1.0, top_p=0.9),
        # a larger vocabulary of odd width in bf16, every request with a setting of its own
        _sample("sample_33x128001_bf16_mixed", 33, 128001, dtype="bf16", mixed=True),
        # the kept distribution for an accept-reject: 32 rows of 9
        _sample("probs_288x49152_p95_m02", 288, 49152, temperature=0.8, top_p=0.95, min_p=0.02, probs=True),
        # one request's tree of 16 in the target
        _commit("commit_b1_n16", 1, 16, 32, 32, 24),
        # 32 requests' trees of 32
        _commit("commit_b32_n32", 32, 32, 32, 32, 24),
    ]


def _attn(name, batch, nodes, ctx, heads, kv, dim=64, dtype="bf16", bs=16, first=0, shared=False, depth=5):
    return {"name": name, "kind": "attn", "batch": batch, "nodes": nodes, "ctx": ctx, "heads": heads, "kv": kv,
            "dim": dim, "dtype": dtype, "bs": bs, "first": first, "shared": shared, "depth": depth}


def _sample(name, rows, vocab, dtype="f32", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, probs=False):
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed, "probs": probs}


def _commit(name, batch, nodes, heads, kv, layers, dim=64, dtype="bf16", bs=16, depth=5, shared=False):
    return {"name": name, "kind": "commit", "batch": batch, "nodes": nodes, "heads": heads, "kv": kv, "layers": layers,
            "dim": dim, "dtype": dtype, "bs": bs, "depth": depth, "shared": shared}


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "sample", "sample", "commit"])
    heads, kv = rng.choice([(32, 32), (9, 3), (32, 8), (8, 1)])
    nodes = _log(rng, 1, 64)
    depth = rng.randint(1, 8)
    if kind == "attn":
        dim = rng.choice([64, 64, 128])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        ctx = _log(rng, 1, 8192)
        most = (1 << 28) // (ctx * kv * dim * 2 * DTYPES[dtype].itemsize)  # no more K/V than the largest listed case
        case = _attn("", _log(rng, 1, max(1, min(32, most))), nodes, ctx, heads, kv, dim, dtype,
                     rng.choice([16, 16, 32, 64, 256]), rng.choice([0, 0, nodes // 2]), rng.random() < 0.3, depth)
    elif kind == "sample":
        vocab = rng.choice([49152, 49152, _log(rng, 1000, 150000), _log(rng, 1000, 150000)])
        case = _sample("", _log(rng, 1, max(1, min(600, 25000000 // vocab))), vocab, rng.choice(["f32", "f32", "bf16"]),
                       round(rng.uniform(0.5, 1.3), 2), rng.choice([0, 0, 20, 50, _log(rng, 1, 400)]),
                       rng.choice([1.0, 0.9, 0.95, round(rng.uniform(0.3, 0.99), 3)]),
                       rng.choice([0.0, 0.0, 0.02, 0.1]), rng.random() < 0.2, rng.random() < 0.3)
    else:
        case = _commit("", _log(rng, 1, 32), nodes, heads, kv, _log(rng, 1, 24), rng.choice([64, 64, 128]),
                       rng.choice(["bf16", "bf16", "f32"]), rng.choice([16, 16, 32, 64]), depth, rng.random() < 0.3)
        if case["dim"] == 128 or case["dtype"] == "f32":
            case["batch"] = min(case["batch"], 8)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs --
def _randn(seed, salt, *shape):
    gen = torch.Generator(device="cuda").manual_seed((seed * 7919 + salt) % (1 << 62))
    return torch.randn(*shape, generator=gen, device="cuda")


def _host_rng(seed, salt):
    return np.random.default_rng([seed % (1 << 62), salt])


def _trees(seed, batch, nodes, depth):
    """parents [batch, nodes] (-1 at node 0) of trees grown level by level, and
    each node's depth and ancestors [batch, nodes, nodes] (itself among them)."""
    rng = _host_rng(seed, 1)
    level = np.zeros(nodes, dtype=np.int64)
    depth = min(depth, nodes - 1)  # a level has a node at least
    level[1:] = 1 + np.arange(nodes - 1) * depth // max(1, nodes - 1)
    starts = np.searchsorted(level, np.arange(depth + 2))
    parents = np.full((batch, nodes), -1, dtype=np.int64)
    for i in range(1, nodes):
        parents[:, i] = rng.integers(starts[level[i] - 1], starts[level[i]], batch)
    above = np.zeros((batch, nodes, nodes), dtype=bool)
    depths = np.zeros((batch, nodes), dtype=np.int64)
    for i in range(nodes):
        above[:, i, i] = True
        if i:
            rows = np.arange(batch)
            above[:, i] |= above[rows, parents[:, i]]
            depths[:, i] = depths[rows, parents[:, i]] + 1
    return parents, depths, above


def _words(above):
    """Ancestors [B, N, N] as bits of int64 words [B, N, ceil(N / 64)]."""
    b, n, _ = above.shape
    words = -(-n // 64)
    padded = np.zeros((b, n, words * 64), dtype=np.uint8)
    padded[:, :, :n] = above
    return np.packbits(padded, axis=2, bitorder="little").view(np.int64)


def _rope(positions, dim):
    inv = 1.0 / THETA ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float32) / dim)
    angle = torch.arange(positions, device="cuda", dtype=torch.float32)[:, None] * inv
    return angle.cos(), angle.sin()


def _pages(seed, state, past, room, most):
    """Block tables for rows that hold past[b] positions (at most `most`) and
    room more, blocks in a random order; returns the pool's number of blocks."""
    bs, batch = state["bs"], state["batch"]
    need = -(-(past + room) // bs)
    ids = _host_rng(seed, 2).permutation(batch * -(-(most + room) // bs) + 3)
    tables = np.zeros((batch, int(need.max())), dtype=np.int32)
    at = 0
    for b in range(batch):
        tables[b, :need[b]] = ids[at:at + need[b]]
        at += need[b]
    state["tables"] = torch.from_numpy(tables).cuda()
    return len(ids)


def prepare(case, seed):
    state = dict(case)
    if case["kind"] == "sample":
        return _prepare_sample(state, seed)
    batch, nodes, heads, kv, dim, bs = (case[k] for k in ("batch", "nodes", "heads", "kv", "dim", "bs"))
    dtype = DTYPES[case["dtype"]]
    parents, depths, above = _trees(seed, 1 if case["shared"] else batch, nodes, case["depth"])
    rng = _host_rng(seed, 3)
    live = np.full(batch, nodes)
    if batch > 1 and not case["shared"]:  # rows whose tree came out smaller
        live[1::3] = np.maximum(1, nodes - 1 - np.arange(batch)[1::3] % max(1, nodes // 4))
    if case["kind"] == "attn":
        past = np.maximum(1, (case["ctx"] * rng.uniform(0.75, 1.0, batch)).astype(np.int64))
        past[0] = case["ctx"]
        blocks = _pages(seed, state, past, case["depth"] + 1, case["ctx"])
        state["k_pool"] = _randn(seed, 10, blocks, kv, bs, dim).to(dtype)
        state["v_pool"] = _randn(seed, 11, blocks, kv, dim, bs).to(dtype)
        # heads from flat to peaked
        sharp = torch.exp(0.5 * _randn(seed, 12, heads, 1)).clamp(0.3, 3.0)
        q = sharp * _randn(seed, 13, batch, nodes, heads, dim)
        rest = _randn(seed, 14, batch, nodes, 2 * kv * dim)
        state["qkv"] = torch.cat([q.flatten(2), rest], 2).to(dtype)
        state["mask"] = torch.from_numpy(_words(above)).cuda()[:, case["first"]:]
        state["seen"] = torch.from_numpy(above).cuda()
        state["depths"] = torch.from_numpy(depths.astype(np.int32)).cuda()
        state["out"] = (0.02 * _randn(seed, 15, batch, nodes - case["first"], heads * dim)).to(dtype)
        state["most"] = int(past.max())
    else:
        past = rng.integers(0, 70, batch)
        accept = _commit_lengths(case)
        blocks = _pages(seed, state, past, case["depth"] + 1, 69)
        layers = case["layers"]
        state["k_pool"] = _randn(seed, 20, layers, blocks, kv, bs, dim).to(dtype)
        state["v_pool"] = _randn(seed, 21, layers, blocks, kv, dim, bs).to(dtype)
        state["qkv"] = _randn(seed, 22, layers, batch, nodes, (heads + 2 * kv) * dim).to(dtype)
        state["seen"] = torch.from_numpy(above).cuda()
        state["parents"] = torch.from_numpy(parents.astype(np.int32)).cuda()
        live[:] = nodes
        # siblings carry different tokens (a node's is its number modulo N), but for
        # a pair now and then; the target samples along the way to a random node as
        # far as the row accepts, and elsewhere what no child carries
        tokens = rng.integers(0, 49152 // nodes, (batch, nodes)) * nodes + np.arange(nodes)
        sampled = rng.integers(0, 49152 // nodes, (batch, nodes)) * nodes + np.arange(nodes)
        for b in range(batch):
            p, a, d = (x[0 if case["shared"] else b] for x in (parents, above, depths))
            deep = np.flatnonzero(d == min(accept[b], d.max()))
            way = np.flatnonzero(a[deep[rng.integers(len(deep))]])
            sampled[b, way[:-1]] = tokens[b, way[1:]]
            if len(way) > 1 and way[1] + 1 < nodes and p[way[1] + 1] == 0:
                tokens[b, way[1] + 1] = tokens[b, way[1]]
        state["tokens"] = torch.from_numpy(tokens).cuda()
        state["sampled"] = torch.from_numpy(sampled).cuda()
        state["room"] = case["depth"] + 1
    state["cos"], state["sin"] = _rope(int(past.max()) + nodes + 1, dim)
    state["meta"] = torch.from_numpy(np.stack([np.arange(batch), past, live]).astype(np.int32)).cuda()
    return state


def _commit_lengths(case):
    """Drafted tokens that each row accepts: 0 .. depth, spread over the rows."""
    return (np.arange(case["batch"]) * 3 + 2) % (min(case["depth"], max(0, case["nodes"] - 1)) + 1)


def _prepare_sample(state, seed):
    rows, vocab = state["rows"], state["vocab"]
    gen = torch.Generator(device="cuda").manual_seed((seed * 7919 + 30) % (1 << 62))
    # a language model's rows: probability falls as a power of the rank, steeper
    # where the context says what comes, over a ranking of the row's own
    rank = torch.rand(rows, vocab, generator=gen, device="cuda").argsort(1).float() + 1
    steep = torch.rand(rows, 1, generator=gen, device="cuda") * 1.8 + 0.9
    logits = 12 - steep * rank.log() + 0.5 * torch.randn(rows, vocab, generator=gen, device="cuda")
    if state["dtype"] == "bf16":
        logits[:, vocab - vocab // 100:] = -math.inf  # ids that pad the vocabulary
    state["logits"] = logits.to(DTYPES[state["dtype"]])
    state["u"] = torch.rand(rows, generator=gen, device="cuda")
    names = ("temperature", "top_k", "top_p", "min_p")
    if state["mixed"]:
        rng = _host_rng(seed, 4)
        per_row = (rng.choice([0.0, 0.6, 0.8, 1.0, 1.2], rows), rng.choice([0, 0, 20, 50, 200], rows),
                   rng.choice([1.0, 1.0, 0.9, 0.95, 0.8], rows), rng.choice([0.0, 0.0, 0.05], rows))
        for name, v in zip(names, per_row):
            state[name] = torch.from_numpy(v.astype(np.int32 if name == "top_k" else np.float32)).cuda()
    return state


# -------------------------------------------------------------- plain form --
def _rotated(x, cos, sin):
    """x [..., heads, dim] in fp32 rotated by cos and sin [..., 1, dim / 2]."""
    x1, x2 = x.chunk(2, -1)
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)


def _plain_attn(s):
    batch, nodes, heads, kv, dim, bs, first = (s[k] for k in ("batch", "nodes", "heads", "kv", "dim", "bs", "first"))
    dtype, dev = s["qkv"].dtype, s["qkv"].device
    past, live = s["meta"][1].long(), s["meta"][2].long()
    at = (past[:, None] + s["depths"])[:, :, None]
    cos, sin = s["cos"][at], s["sin"][at]
    q, k, v = s["qkv"].split([heads * dim, kv * dim, kv * dim], 2)
    q = _rotated(q.view(batch, nodes, heads, dim).float(), cos, sin).to(dtype).float()[:, first:]
    k = _rotated(k.view(batch, nodes, kv, dim).float(), cos, sin).to(dtype).float()
    v = v.view(batch, nodes, kv, dim).float()
    # the cached keys and values of each row, in order, then the tree's
    pages = s["tables"][s["meta"][0].long(), :-(-s["most"] // bs)].long()
    old_k = s["k_pool"][pages].permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, dim).float()
    old_v = s["v_pool"][pages].permute(0, 2, 1, 4, 3).reshape(batch, kv, -1, dim).float()
    k = torch.cat([old_k, k.transpose(1, 2)], 2)
    v = torch.cat([old_v, v.transpose(1, 2)], 2)
    rows = (nodes - first) * (heads // kv)
    q = q.view(batch, nodes - first, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv, rows, dim)
    cached = old_k.shape[2]
    see_old = (torch.arange(cached, device=dev) < past[:, None])[:, None].expand(batch, nodes - first, cached)
    see_new = s["seen"][:, first:] & (torch.arange(nodes, device=dev) < live[:, None])[:, None]
    see = torch.cat([see_old, see_new], 2).repeat_interleave(heads // kv, 1)[:, None]
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * dim ** -0.5
    score = score.masked_fill(~see, -math.inf)
    weight = torch.exp(score - score.amax(3, keepdim=True))
    o = torch.matmul(weight, v) / weight.sum(3, keepdim=True)
    o = o.view(batch, kv, nodes - first, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(batch, nodes - first, -1)
    written = (torch.arange(first, nodes, device=dev) < live[:, None])[:, :, None]
    s["out"].copy_(torch.where(written, o.to(dtype), s["out"]))
    return s["out"]


def _column(v, dev, dtype):
    """A parameter as fp32 (int32) holds it, as a column in 64 bits."""
    if isinstance(v, torch.Tensor):
        return v[:, None].to(dtype)
    return torch.tensor([[v]], dtype=torch.float32, device=dev).to(dtype)


def _plain_sample(s):
    x, u = s["logits"].double(), s["u"].double()[:, None]
    rows, vocab = x.shape
    temperature, top_p, min_p = (_column(s[k], x.device, torch.float64) for k in ("temperature", "top_p", "min_p"))
    top_k = _column(s["top_k"], x.device, torch.int64)
    top_k = torch.where(temperature > 0, torch.where(top_k > 0, top_k, vocab), 1)
    x = torch.where(x.isnan(), -math.inf, x)
    w = torch.exp((x - x.amax(1, keepdim=True)) / torch.where(temperature > 0, temperature, 1.0))
    down, ids = torch.sort(w, dim=1, descending=True, stable=True)
    # ties of the logits, not of the weights: both orders are the same but where weights underflow
    rank = torch.arange(vocab, device=x.device)[None]
    among = torch.where(rank < top_k, down, 0.0)
    mass = among.cumsum(1)
    total = mass[:, -1:]
    kept = (rank < top_k) & ((down >= min_p) | (rank == 0)) & ((mass - among < top_p * total) | (top_p >= 1) | (rank == 0))
    down = torch.where(kept, down, 0.0)
    w = torch.zeros_like(w).scatter_(1, ids, down)
    run = w.cumsum(1)
    token = (run <= u * run[:, -1:]).sum(1).clamp_max(vocab - 1)
    return (token, (w / run[:, -1:]).float()) if s["probs"] else token


def _plain_commit(s):
    batch, nodes, heads, kv, dim, bs = (s[k] for k in ("batch", "nodes", "heads", "kv", "dim", "bs"))
    dev = s["qkv"].device
    row, past, live = s["meta"].long()
    parents = s["parents"].long().expand(batch, nodes)
    seen = s["seen"].expand(batch, nodes, nodes)
    node = torch.arange(nodes, device=dev)
    # a node is on the way if the target sampled it and every ancestor of it, the
    # lowest of the siblings that carry the token
    hit = (s["tokens"] == s["sampled"].gather(1, parents.clamp_min(0))) & (node > 0) & (node < live[:, None])
    same = (parents[:, :, None] == parents[:, None]) & (s["tokens"][:, :, None] == s["tokens"][:, None])
    hit &= ~(same & (node[None] < node[:, None])).any(2)
    on = ~(seen & ~(hit | (node == 0))[:, None]).any(2)
    on &= seen.sum(2) <= s["room"]
    n = on.sum(1) - 1
    path = torch.where(on, node, nodes).sort(1).values
    kept = path < nodes
    at = path.clamp_max(nodes - 1)
    last = at.gather(1, n[:, None])
    drafted = torch.where(kept, s["tokens"].gather(1, at), -1)[:, 1:]
    verdict = torch.cat([n[:, None], s["sampled"].gather(1, last), drafted], 1).t().contiguous()
    b, j = kept.nonzero(as_tuple=True)
    position = past[b] + j
    block, slot = s["tables"][row[b], position // bs].long(), position % bs
    _, k, v = s["qkv"][:, b, at[b, j]].split([heads * dim, kv * dim, kv * dim], 2)
    cos, sin = s["cos"][position][None, :, None], s["sin"][position][None, :, None]
    k = _rotated(k.view(k.shape[0], -1, kv, dim).float(), cos, sin).to(s["qkv"].dtype)
    s["k_pool"][:, block, :, slot] = k.transpose(0, 1)
    s["v_pool"][:, block, :, :, slot] = v.view(v.shape[0], -1, kv, dim).transpose(0, 1)
    return verdict, torch.where(kept, path, -1).int(), s["k_pool"], s["v_pool"]


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "sample": _plain_sample, "commit": _plain_commit}[state["kind"]](state)


def work(case):
    kind = case["kind"]
    size = DTYPES[case["dtype"]].itemsize
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + (4 * n if case["probs"] else 0) + 12 * case["rows"], "flops": 6 * n}
    batch, nodes, heads, kv, dim = (case[k] for k in ("batch", "nodes", "heads", "kv", "dim"))
    if kind == "attn":
        queries = nodes - case["first"]
        keys = batch * 0.875 * case["ctx"] if batch > 1 else case["ctx"]
        moved = 2 * keys * kv * dim + batch * (queries * 2 * heads * dim + nodes * 2 * kv * dim)
        return {"bytes": int(moved * size), "flops": int(4 * queries * heads * dim * (keys + batch * case["depth"]))}
    tokens = int(_commit_lengths(case).sum()) + batch
    return {"bytes": 2 * case["layers"] * tokens * 2 * kv * dim * size + 20 * batch * nodes,
            "flops": 3 * case["layers"] * tokens * kv * dim}


# --------------------------------------------------------------- 64 bits ----
def _turned(x, cos, sin):
    """x [n, heads, dim] rotated in 64 bits by the angles' cos and sin [n, dim / 2], then as its type holds it."""
    half = x.shape[2] // 2
    a, b = x[:, :, :half].double(), x[:, :, half:].double()
    c, d = cos[:, None].double(), sin[:, None].double()
    return torch.cat([a * c - b * d, b * c + a * d], 2).to(x.dtype).double()


def _exact_attn(s):
    heads, kv, dim, bs, first = (s[k] for k in ("heads", "kv", "dim", "bs", "first"))
    out = s["out"].double()
    for b in range(s["batch"]):
        row, past, live = s["meta"][:, b].tolist()
        tree = 0 if s["shared"] else b
        if live <= first:
            continue
        at = past + s["depths"][tree, :live].long()
        x = s["qkv"][b, :live].view(live, heads + 2 * kv, dim)
        q = _turned(x[first:, :heads], s["cos"][at[first:]], s["sin"][at[first:]])
        k = _turned(x[:, heads:heads + kv], s["cos"][at], s["sin"][at])
        ids = s["tables"][row, :-(-past // bs)].long()
        for h in range(kv):
            mine = slice(h * (heads // kv), (h + 1) * (heads // kv))
            keys = torch.cat([s["k_pool"][ids, h].reshape(-1, dim)[:past].double(), k[:, h]])
            values = torch.cat([s["v_pool"][ids, h].transpose(1, 2).reshape(-1, dim)[:past].double(),
                                x[:, heads + kv + h].double()])
            z = torch.einsum("ngd,kd->gnk", q[:, mine], keys) / math.sqrt(dim)
            z[:, :, past:][:, ~s["seen"][tree, first:live, :live]] = -math.inf
            o = torch.softmax(z, 2) @ values
            out[b, :live - first].view(live - first, heads, dim)[:, mine] = o.transpose(0, 1)
    return out


def _exact_sample(s):
    tokens, probs = [], []
    for r in range(s["rows"]):
        t, k, p, m = (float(s[n][r]) if isinstance(s[n], torch.Tensor) else float(np.float32(s[n]))
                      for n in ("temperature", "top_k", "top_p", "min_p"))
        x = s["logits"][r].double()
        ids = torch.argsort(x, descending=True, stable=True)
        if t == 0:
            ids = ids[:1]
        elif k > 0:
            ids = ids[:int(k)]
        w = ((x[ids] - x[ids[0]]) / (t or 1.0)).exp()
        mass = w.cumsum(0)
        keep = len(ids) if p >= 1 else min(len(ids), int((mass < p * mass[-1]).sum()) + 1)
        keep = max(1, min(keep, int((w >= m).sum())))
        row = torch.zeros_like(x)
        row[ids[:keep]] = w[:keep] / w[:keep].sum()
        run = row.cumsum(0)
        tokens.append(min(len(x) - 1, int(torch.searchsorted(run, s["u"][r].double() * run[-1], right=True))))
        probs.append(row)
    token = torch.tensor(tokens, device=s["logits"].device)
    return (token, torch.stack(probs)) if s["probs"] else token


def _exact_commit(s):
    heads, kv, dim, bs, nodes = (s[k] for k in ("heads", "kv", "dim", "bs", "nodes"))
    tokens, sampled, meta, tables = (s[k].tolist() for k in ("tokens", "sampled", "meta", "tables"))
    parents = s["parents"].expand(s["batch"], nodes).tolist()
    verdicts, paths = [], []
    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    for b in range(s["batch"]):
        way = [0]
        while len(way) < s["room"]:
            child = [c for c in range(way[-1] + 1, meta[2][b])
                     if parents[b][c] == way[-1] and tokens[b][c] == sampled[b][way[-1]]]
            if not child:
                break
            way.append(child[0])
        fill = [-1] * (nodes - len(way))
        verdicts.append([len(way) - 1, sampled[b][way[-1]]] + [tokens[b][c] for c in way[1:]] + fill)
        paths.append(way + fill)
        for j, c in enumerate(way):
            at = meta[1][b] + j
            block, slot = tables[meta[0][b]][at // bs], at % bs
            x = s["qkv"][:, b, c].view(-1, heads + 2 * kv, dim)
            turn = [t[at].expand(len(x), dim // 2) for t in (s["cos"], s["sin"])]
            k_pool[:, block, :, slot] = _turned(x[:, heads:heads + kv], *turn)
            v_pool[:, block, :, :, slot] = x[:, heads + kv:].double()
    dev = s["qkv"].device
    return (torch.tensor(verdicts, device=dev).t().contiguous(), torch.tensor(paths, dtype=torch.int32, device=dev),
            k_pool, v_pool)


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "sample": _exact_sample, "commit": _exact_commit}[s["kind"]](s)


# ------------------------------------------------------ the framework's own --
_ops = None


def _run_own(s):
    global _ops
    if _ops is None:
        package = str(Path(__file__).resolve().parent.parent / "speculative-decoder_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from specdec import ops as _ops
    kind = s["kind"]
    if kind == "sample":
        probs = torch.empty(s["rows"], s["vocab"], device="cuda") if s["probs"] else None
        token = _ops.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], probs=probs)
        return (token, probs) if s["probs"] else token
    if kind == "attn":
        return _ops.tree_attention(s["qkv"], s["cos"], s["sin"], s["k_pool"], s["v_pool"], s["tables"], s["meta"],
                                   s["mask"], s["depths"], s["heads"], s["dim"] ** -0.5, s["most"], first=s["first"],
                                   out=s["out"])
    verdict, path = _ops.tree_commit(s["tokens"], s["parents"], s["sampled"], s["meta"], s["room"], s["qkv"], s["cos"],
                                     s["sin"], s["k_pool"], s["v_pool"], s["tables"])
    return verdict, path, s["k_pool"], s["v_pool"]
