"""Trees of drafted tokens as the tree operators read them.

A tree has N nodes a row, parents before children; node 0 is the last token of
the context, whose keys and values the cache does not hold yet.  No counterpart
in the reference, which drafts a chain (spec/draft.py).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from specdec import ops


def plan(parents: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(mask, depth) of parents [B, N] (any integer type, -1 for node 0), on
    their device: mask int64 [B, N, ceil(N / 64)], a bit for each node's ancestors
    and itself (bit j % 64 of word j / 64), depth int32 [B, N], its distance from
    node 0.  A parent that does not come before its child is an error on the
    host, where the tree is; on a GPU the caller answers for it."""
    if parents.dim() != 2 or parents.shape[1] == 0:
        raise ValueError(f"parents must be [B, N] with a node 0 (got {list(parents.shape)})")
    b, n = parents.shape
    node = torch.arange(n, device=parents.device)
    up = parents.long()
    if not parents.is_cuda and bool(((up >= node) | (up < -1) | ((up < 0) != (node == 0))).any()):
        raise ValueError("node 0 is the root (-1); every other node's parent comes before it")
    up = up.clamp_min(0)
    words = -(-n // 64)
    bit = torch.ones((), dtype=torch.int64, device=parents.device) << (node % 64)
    mask = torch.where(node[:, None] // 64 == torch.arange(words, device=parents.device), bit[:, None], 0).expand(b, n, words)
    depth = (node > 0).long().expand(b, n)
    # a node's ancestors are those in reach of 1, 2, 4, .. steps, and its reach's reach
    for _ in range(max(1, (n - 1).bit_length())):
        mask = mask | mask.gather(1, up[:, :, None].expand(b, n, words))
        depth = depth + depth.gather(1, up)
        up = up.gather(1, up)
    return mask.contiguous(), depth.int()


@dataclass(frozen=True)
class TreeStep:
    """What a forward over tree nodes needs beside a chain's: the masks int64 [B
    or 1, N - first, ..] of the nodes that it runs, first .. N - 1, the depths
    int32 [B or 1, N] of all, and `qkv` [layers, B, N, ..], where each layer's
    projections of the nodes are kept for the levels after them and for the
    commit.  `past` bounds the rows' cached lengths."""

    mask: torch.Tensor
    depth: torch.Tensor
    qkv: torch.Tensor
    past: int
    first: int = 0

    @staticmethod
    def store(llama, batch: int, nodes: int) -> torch.Tensor:
        """An empty `qkv` for `nodes` nodes of `batch` rows."""
        cfg = llama.config
        row = (cfg.num_attention_heads + 2 * cfg.num_key_value_heads) * cfg.head_dim
        return torch.empty(len(llama.layers), batch, nodes, row, dtype=llama.embed.dtype, device=llama.embed.device)

    def attend(self, layer: int, qkv: torch.Tensor, llama, cache, meta: torch.Tensor, out: torch.Tensor) -> None:
        """The attention of this step's nodes in one layer, from their
        projections qkv [B, N - first, ..], into out."""
        kept = self.qkv[layer]
        kept[:, self.first:].copy_(qkv)
        ops.tree_attention(kept, llama.rope_cos, llama.rope_sin, cache.k[layer], cache.v[layer], cache.table_tensor, meta,
                           self.mask, self.depth, llama.config.num_attention_heads, llama.scaling, self.past, self.first,
                           out)
