"""Speculative decoding of a tree of drafted tokens a round.

No counterpart in the reference, whose rounds draft a chain (spec/loop.py).  A
drafter proposes a tree whose node 0 is the context's last token; the target
runs all nodes in one forward (ops.tree_attention), a token is drawn from the
target's restricted distribution at every node (ops.sample), and the walk down
the tree follows the drawn tokens as long as a child carries them
(ops.tree_commit, which appends the walked path's keys and values to the cache
in the same launch).  Each emitted token is a draw from the target at its own
context, whatever was drafted, so the output is distributed as plain decoding's
(at temperature 0 it is the target's greedy decoding, up to the rounding of
logits that tie within the batch sizes' different sums).
"""
from __future__ import annotations

from collections.abc import Callable
from dataclasses import dataclass, field
from typing import Protocol

import torch

from cache.kv import KVCache
from lm import tree as trees
from lm.forward import forward_core
from lm.model import as_llama
from lm.sampling import draw
from lm.tree import TreeStep
from specdec import ops
from spec.draft import run
from spec.loop import _cut, _release, _Request


class TreeDrafter(Protocol):
    def prefill(self, seq_ids: list[int], prompts: list[list[int]]) -> None: ...

    def propose(self, seq_ids: list[int], contexts: list[list[int]]) -> tuple[torch.Tensor, torch.Tensor]:
        """Returns tokens int64 [B, N], node 0 each context's last token, and
        parents [B or 1, N] on the host, -1 for node 0 and before its child for
        every other node."""
        ...

    def rollback(self, seq_id: int, keep: int) -> None: ...

    def release(self, seq_id: int) -> None: ...


@dataclass
class TreeStats:
    """rounds run; drafted and accepted nodes, and the tokens emitted, summed over the rows."""

    rounds: int = 0
    drafted: int = 0
    accepted: int = 0
    emitted_per_round: list[int] = field(default_factory=list)


def tree_shape(branching: list[int]) -> torch.Tensor:
    """parents int32 [1, N] of the tree whose nodes of level l have branching[l] children each."""
    parents, level = [-1], [0]
    for width in branching:
        if width < 1:
            raise ValueError(f"a level has at least one child a node (got {branching})")
        children = [p for p in level for _ in range(width)]
        level = list(range(len(parents), len(parents) + len(children)))
        parents += children
    if len(parents) > ops.TREE_NODES:
        raise ValueError(f"a tree has at most {ops.TREE_NODES} nodes (got {len(parents)})")
    return torch.tensor([parents], dtype=torch.int32)


class ModelTree:
    """A draft model's likeliest continuations: the nodes of level l carry the
    branching[l] likeliest tokens after their parent.  Each level but the last
    is one forward of its nodes over the draft's cache and the levels before it;
    none of it enters the draft's cache, which holds the context alone."""

    def __init__(self, model, cache: KVCache, branching: list[int]) -> None:
        if not branching:
            raise ValueError("a tree to draft has a level at least (got none)")
        self.model, self.cache, self.branching = model, cache, list(branching)
        self.parents = tree_shape(self.branching)
        mask, depth = trees.plan(self.parents)
        # the drafted nodes by themselves: node 0 is in the draft's cache
        n = self.parents.shape[1] - 1
        bits = (mask[..., None] >> torch.arange(64)) & 1
        bits = torch.nn.functional.pad(bits.flatten(2)[:, 1:, 1:1 + n], (0, -n % 64)).view(1, n, -1, 64)
        self._mask = (bits << torch.arange(64)).sum(-1).to(cache.device)
        self._depth = (depth[:, 1:] - 1).contiguous().to(cache.device)

    def prefill(self, seq_ids: list[int], prompts: list[list[int]]) -> None:
        for seq_id in seq_ids:
            self.cache.add(seq_id)
        run(self.model, self.cache, seq_ids, prompts)

    def propose(self, seq_ids: list[int], contexts: list[list[int]]) -> tuple[torch.Tensor, torch.Tensor]:
        cache, b = self.cache, len(seq_ids)
        llama = as_llama(self.model, cache.device)
        pending = [ctx[cache.length(s):] for s, ctx in zip(seq_ids, contexts)]
        logits = run(self.model, cache, seq_ids, pending)
        nodes = self.parents.shape[1] - 1
        lengths = [cache.length(s) for s in seq_ids]
        llama.ensure_positions(max(lengths) + len(self.branching) + 1)
        rows = [cache.tables[s].row for s in seq_ids]
        meta = torch.tensor([rows, lengths, [nodes] * b], dtype=torch.int32).to(cache.device, non_blocking=True)
        kept = TreeStep.store(llama, b, nodes)
        last = torch.tensor([[ctx[-1]] for ctx in contexts], dtype=torch.int64).to(cache.device, non_blocking=True)
        tokens, start = [last], 0
        for level, width in enumerate(self.branching):
            ids = torch.topk(logits, width, dim=-1).indices.view(b, -1)
            tokens.append(ids)
            end = start + ids.shape[1]
            if level + 1 < len(self.branching):
                words = -(-end // 64)
                step = TreeStep(self._mask[:, start:end, :words].contiguous(), self._depth[:, :end].contiguous(),
                                kept[:, :, :end], max(lengths), start)
                logits = forward_core(llama, cache, meta, ids, max(lengths), tree=step)
            start = end
        return torch.cat(tokens, dim=1), self.parents

    def rollback(self, seq_id: int, keep: int) -> None:
        self.cache.truncate(seq_id, min(self.cache.length(seq_id), keep))

    def release(self, seq_id: int) -> None:
        self.cache.free(seq_id)


@torch.no_grad()
def verify_tree(target, cache: KVCache, seq_ids: list[int], contexts: list[list[int]], tokens: torch.Tensor,
                parents: torch.Tensor, u: torch.Tensor, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """One target forward over the rows' trees, a draw at every node and the
    commit of each row's path: the verdict of ops.tree_commit, int64 [N + 1, B],
    on the GPU.  tokens int64 [B, N]; parents [B or 1, N] on the host; u fp32 [B,
    N].  The cache holds the contexts but their last tokens on entry, and room
    for each row's longest path on return: the caller truncates it to the past
    and the n + 1 nodes that the verdict keeps.  A call that raises leaves its
    lengths as they were."""
    for seq_id, ctx in zip(seq_ids, contexts):
        if cache.length(seq_id) != len(ctx) - 1:
            raise RuntimeError(f"seq {seq_id}: target cache holds {cache.length(seq_id)}, expected {len(ctx) - 1}")
    b = len(seq_ids)
    if tokens.dim() != 2 or tokens.shape[0] != b or len(contexts) != b or not 0 < tokens.shape[1] <= ops.TREE_NODES:
        raise ValueError(f"tokens must be [{b}, N] of at most {ops.TREE_NODES} nodes for {len(contexts)} contexts "
                         f"(got {list(tokens.shape)})")
    n = tokens.shape[1]
    if len(set(seq_ids)) != b:
        raise ValueError(f"each sequence is verified once a call (got {list(seq_ids)})")
    if parents.dim() != 2 or parents.shape[0] not in (1, b) or parents.shape[1] != n:
        raise ValueError(f"parents must be [{b} or 1, {n}] (got {list(parents.shape)})")
    if u.numel() != b * n:
        raise ValueError(f"u must be [{b}, {n}], a uniform a node (got {list(u.shape)})")
    llama = as_llama(target, cache.device)
    mask, depth = trees.plan(parents)
    room = int(depth.max()) + 1
    try:
        step = cache.append(seq_ids, [room] * b, nodes=[n] * b)
        llama.ensure_positions(step.max_total)
        tokens = tokens.to(cache.device, torch.int64)
        up = parents.to(torch.int32).to(cache.device, non_blocking=True)
        past = max(step.past)
        tree = TreeStep(mask.to(cache.device, non_blocking=True), depth.to(cache.device, non_blocking=True),
                        TreeStep.store(llama, b, n), past)
        logits = forward_core(llama, cache, step.meta, tokens, past, tree=tree)
        sampled = draw(logits, u, temperature, top_k, top_p, min_p)
        verdict, _ = ops.tree_commit(tokens, up, sampled, step.meta, room, tree.qkv, llama.rope_cos, llama.rope_sin, cache.k,
                                     cache.v, cache.table_tensor)
    except Exception:
        # rows that have grown, too few blocks for the rest among the reasons
        for seq_id, ctx in zip(seq_ids, contexts):
            cache.truncate(seq_id, len(ctx) - 1)
        raise
    return verdict


def _drawn(req: _Request, n: int, tokens: list[int]) -> None:
    """Raises for a row that has no token to go on with, which a next forward would
    look up as id -1: its logits hold no number (ops.sample), or its path no slot
    (ops.tree_commit, n = -1)."""
    if n < 0 or tokens[-1] < 0:
        raise RuntimeError(f"seq {req.seq_id}: no token after {len(req.context)} tokens; the target's logits there are "
                           "no numbers, or the cache has no slot for them")


@torch.no_grad()
def generate_tree(target, cache: KVCache, drafter: TreeDrafter, prompts: list[list[int]], max_new_tokens: int,
                  temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0,
                  generator: torch.Generator | None = None, eos_id: int | None = None,
                  on_event: Callable[[str], None] | None = None) -> tuple[list[list[int]], TreeStats]:
    """Speculative decoding of `prompts` with `drafter`'s trees; returns each
    prompt's new tokens and the statistics.  Every token is a draw from the
    target's distribution under temperature, top-k, top-p and min-p, with
    uniforms from `generator`: one a row for the first token, then one a node
    and round.  A row whose logits hold no number is an error.  Events as
    `spec.loop.generate`'s."""
    gen = generator if generator is not None else torch.Generator().manual_seed(0)
    event = on_event if on_event is not None else (lambda name: None)
    stats = TreeStats()
    requests = [_Request(i, list(p)) for i, p in enumerate(prompts)]
    seq_ids = [r.seq_id for r in requests]
    uniforms = lambda *shape: torch.rand(*shape, generator=gen, dtype=torch.float32, device=gen.device)
    for s in seq_ids:
        cache.add(s)
    logits = run(target, cache, seq_ids, prompts)
    firsts = draw(logits, uniforms(len(prompts)), temperature, top_k, top_p, min_p).tolist()
    event("first_token")
    for req, token in zip(requests, firsts):
        _drawn(req, 0, [token])
    drafter.prefill(seq_ids, [r.context for r in requests])
    event("draft_prefilled")
    live = []
    for req, token in zip(requests, firsts):
        req.extend([token])
        if req.done(max_new_tokens, eos_id):
            _release(cache, drafter, req.seq_id)
        else:
            live.append(req)

    while live:
        ids = [r.seq_id for r in live]
        contexts = [r.context for r in live]
        tokens, parents = drafter.propose(ids, contexts)
        verdict = verify_tree(target, cache, ids, contexts, tokens, parents, uniforms(*tokens.shape), temperature, top_k,
                              top_p, min_p).t().tolist()  # the round's one copy to the host
        stats.rounds += 1
        survivors = []
        for req, (n, after, *drafted) in zip(live, verdict):
            kept = _cut(drafted[:n] + [after], max_new_tokens - len(req.output), eos_id)
            _drawn(req, n, kept)
            stats.drafted += tokens.shape[1] - 1
            stats.accepted += n
            stats.emitted_per_round.append(len(kept))
            before = len(req.context)
            req.extend(kept)
            if req.done(max_new_tokens, eos_id):
                _release(cache, drafter, req.seq_id)
            else:
                cache.truncate(req.seq_id, before + n)
                drafter.rollback(req.seq_id, before + n)
                survivors.append(req)
        live = survivors
        if stats.rounds == 1:
            event("first_round")
    return [r.output for r in requests], stats
