"""Rounds of trees: what each emitted token was drawn with, and what a round that
fails leaves behind."""
import pytest
import torch

import spec.tree as rounds
import tree_ref
from cache.kv import KVCache
from lm.forward import forward
from lm.sampling import draw
from spec.tree import ModelTree, generate_tree, tree_shape, verify_tree
from tiny_models import early_exit, random_prompts, tiny64

pytestmark = pytest.mark.gpu


def cache_for(model, dtype=torch.float32, blocks=128, bs=16):
    return KVCache.for_model(model.config, blocks, bs, dtype, "cuda")


def test_logits_that_are_no_numbers_end_the_rounds(monkeypatch):
    """From the first token on, and from the second round on; nothing is looked up after them."""
    target = tiny64(0)
    prompts = random_prompts(2, 256, 17)
    for good in (0, 2):  # draws before the logits turn into NaN
        drafter = ModelTree(early_exit(target), cache_for(early_exit(target)), [2, 1])
        calls = []

        def spoiled(logits, *a):
            calls.append(len(calls))
            return draw(logits if calls[-1] < good else logits * float("nan"), *a)

        monkeypatch.setattr(rounds, "draw", spoiled)
        with pytest.raises(RuntimeError, match="no token"):
            generate_tree(target, cache_for(target), drafter, prompts, 9, temperature=0.8)
        assert len(calls) == good + 1
    torch.cuda.synchronize()
