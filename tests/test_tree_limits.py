"""What the tree operators and the sampler refuse before any launch (no GPU
needed), and the trees and definitions that their GPU tests are written with."""
import ctypes

import numpy as np
import pytest
import torch

from specdec import _lib, ops
from tree_ref import Case, ancestors, draw, random_parents, walk, words

FAKE = 1 << 20  # never read: each call below returns before a launch
OK, EINVAL, EUNSUPPORTED = 0, 1, 3


def attention(**kw):
    a = dict(qkv=FAKE, dtype=2, batch_stride=12 * 512, token_stride=512, cos=FAKE, sin=FAKE, positions=100, k=FAKE,
             v=FAKE, blocks=8, tables=FAKE, table_stride=4, table_rows=2, table_cols=4, meta=FAKE, mask=FAKE,
             mask_batch=12, mask_row=1, depth=FAKE, depth_batch=12, batch=2, nodes=12, first=0, heads=4, kv=2, dim=64,
             bs=16, scale=0.125, most=64, ws=None, floats=0, out=FAKE, out_batch=12 * 256, out_token=256, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().specdec_tree_attention(*a.values())


@pytest.mark.parametrize("change", [
    dict(batch=-1), dict(nodes=-1), dict(first=-1), dict(first=13), dict(heads=0), dict(kv=0), dict(heads=3),
    dict(bs=0), dict(positions=0), dict(blocks=-1), dict(table_rows=-1), dict(table_cols=-1), dict(table_stride=3),
    dict(most=-1), dict(floats=-1), dict(token_stride=511), dict(out_token=255), dict(qkv=None), dict(cos=None),
    dict(sin=None), dict(k=None), dict(v=None), dict(tables=None), dict(meta=None), dict(mask=None), dict(depth=None),
    dict(out=None)])
def test_attention_refuses_invalid_arguments(change):
    assert attention(**change) == EINVAL


@pytest.mark.parametrize("change", [dict(dim=32), dict(dim=96), dict(dim=256), dict(dtype=1), dict(nodes=257, first=0),
                                    dict(batch=65536), dict(blocks=1 << 31), dict(positions=1 << 31)])
def test_attention_refuses_what_it_does_not_implement(change):
    assert attention(**change) == EUNSUPPORTED


def test_attention_of_nothing_launches_nothing():
    assert attention(batch=0) == OK and attention(first=12) == OK and attention(nodes=0) == OK


def test_attention_workspace_needs_no_gpu():
    lib, floats = _lib.load(), ctypes.c_int64(-1)
    assert lib.specdec_tree_attention_workspace(2, 12, 0, 4, 2, 64, 2, 16, 4096, ctypes.byref(floats)) == OK
    assert floats.value >= 0
    assert lib.specdec_tree_attention_workspace(-1, 12, 0, 4, 2, 64, 2, 16, 4096, ctypes.byref(floats)) == EINVAL
    assert lib.specdec_tree_attention_workspace(2, 12, 13, 4, 2, 64, 2, 16, 4096, ctypes.byref(floats)) == EINVAL
    assert lib.specdec_tree_attention_workspace(2, 12, 0, 4, 2, 64, 2, 16, 4096, None) == EINVAL


def commit(**kw):
    a = dict(tokens=FAKE, tokens_stride=12, parents=FAKE, parents_stride=12, sampled=FAKE, sampled_stride=12, meta=FAKE,
             batch=2, nodes=12, room=6, verdict=FAKE, path=FAKE, qkv=FAKE, dtype=2, layers=3, layer_stride=2 * 12 * 512,
             batch_stride=12 * 512, token_stride=512, cos=FAKE, sin=FAKE, positions=100, heads=4, kv=2, dim=64, bs=16,
             k=FAKE, v=FAKE, blocks=8, tables=FAKE, table_stride=4, table_rows=2, table_cols=4, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().specdec_tree_commit(*a.values())


@pytest.mark.parametrize("change", [
    dict(batch=-1), dict(nodes=0), dict(room=0), dict(layers=-1), dict(tokens=None), dict(parents=None),
    dict(sampled=None), dict(meta=None), dict(verdict=None), dict(path=None), dict(qkv=None), dict(cos=None),
    dict(sin=None), dict(k=None), dict(v=None), dict(tables=None), dict(kv=0), dict(bs=0), dict(dim=0),
    dict(positions=0), dict(blocks=0), dict(table_rows=0), dict(table_cols=0), dict(table_stride=3),
    dict(token_stride=511)])
def test_commit_refuses_invalid_arguments(change):
    assert commit(**change) == EINVAL


@pytest.mark.parametrize("change", [dict(nodes=257), dict(dim=33), dict(dim=514, token_stride=8 * 514), dict(dtype=1), dict(layers=65536),
                                    dict(blocks=1 << 31), dict(positions=1 << 31)])
def test_commit_refuses_what_it_does_not_implement(change):
    assert commit(**change) == EUNSUPPORTED


def test_commit_of_nothing_launches_nothing():
    assert commit(batch=0) == OK


def sampler(**kw):
    a = dict(logits=FAKE, dtype=0, rows=3, vocab=100, stride=100, u=FAKE, t=1.0, ts=None, k=0, ks=None, p=1.0, ps=None,
             m=0.0, ms=None, token=FAKE, probs=None, probs_stride=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().specdec_sample(*a.values())


def test_sampler_limits():
    for change in (dict(rows=-1), dict(vocab=0), dict(stride=99), dict(logits=None), dict(u=None), dict(token=None),
                   dict(probs=FAKE, probs_stride=99)):
        assert sampler(**change) == EINVAL, change
    for change in (dict(dtype=1), dict(vocab=(1 << 24) + 1, stride=1 << 25), dict(rows=1 << 31)):
        assert sampler(**change) == EUNSUPPORTED, change
    assert sampler(rows=0) == OK


def test_wrappers_refuse_host_tensors():
    case = Case(0, [5], 3, 2, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        case.call(ops, dev="cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        ops.sample(torch.randn(2, 8), torch.rand(2))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.tree_commit(torch.zeros(1, 3, dtype=torch.int64), case.parents, torch.zeros(1, 3, dtype=torch.int64), case.meta)


def test_reference_trees():
    parents = torch.tensor([[-1, 0, 0, 1, 3]])
    seen, depth = ancestors(parents)
    assert depth.tolist() == [[0, 1, 1, 2, 3]]
    assert words(seen)[0, :, 0].tolist() == [1, 3, 5, 11, 27]
    wide = ancestors(random_parents(np.random.default_rng(0), 2, 70))[0]
    bits = words(wide)
    assert bits.shape == (2, 70, 2)
    for j in (0, 63, 64, 69):
        assert torch.equal(bits[:, :, j // 64] >> (j % 64) & 1, wide[:, :, j].long())
    # the lowest of two children that carry the token; nothing past the room or the live nodes
    tokens, sampled = [9, 4, 4, 7, 7], [4, 7, 7, 7, 1]
    assert walk(tokens, parents[0], sampled, 5, 5) == [0, 1, 3, 4]
    assert walk(tokens, parents[0], sampled, 4, 5) == [0, 1, 3] and walk(tokens, parents[0], sampled, 5, 2) == [0, 1]
    assert walk(tokens, parents[0], sampled, 0, 5) == []


def test_reference_draws():
    x = torch.tensor([1.0, 3.0, 3.0, 2.0, float("-inf")])
    e = [float(v) for v in torch.exp(torch.tensor([-2.0, 0.0, 0.0, -1.0], dtype=torch.float64))]
    token, p, _ = draw(x, 0.0, 1.0, 0, 1.0, 0.0)
    assert token == 0 and abs(float(p[0]) - e[0] / sum(e)) < 1e-15 and float(p[4]) == 0
    assert draw(x, 0.999, 1.0, 0, 1.0, 0.0)[0] == 3
    assert draw(x, 0.999, 0.0, 0, 1.0, 0.0)[0] == 1  # greedy: the lower of a tie
    assert draw(x, 0.999, 1.0, 1, 1.0, 0.0)[0] == 1 and draw(x, 0.6, 1.0, 2, 1.0, 0.0)[0] == 2
    assert (draw(x, 0.5, 1.0, 0, 0.5, 0.0)[1] > 0).tolist() == [False, True, True, False, False]
    assert (draw(x, 0.5, 1.0, 0, 1.0, 0.3)[1] > 0).tolist() == [False, True, True, True, False]
    assert draw(torch.full((3,), float("nan")), 0.5, 1.0, 0, 1.0, 0.0)[0] == -1


@pytest.mark.parametrize("nodes", [1, 2, 3, 31, 64, 65, 256])
def test_plan_of_a_tree(nodes):
    from lm import tree

    for reach in (1, 3, None):  # a chain, deep trees, shallow ones
        parents = random_parents(np.random.default_rng(nodes), 3, nodes, reach)
        mask, depth = tree.plan(parents)
        seen, want = ancestors(parents)
        assert torch.equal(mask, words(seen)) and torch.equal(depth, want)


def test_plan_refuses_what_is_no_tree():
    from lm import tree

    for rows in ([[0]], [[-1, 1]], [[-1, 2, 0]], [[-1, -1]], [[-1, -2]], [[0, 0]]):
        with pytest.raises(ValueError):
            tree.plan(torch.tensor(rows))
    for shape in ((0,), (2, 0)):
        with pytest.raises(ValueError):
            tree.plan(torch.zeros(shape, dtype=torch.int32))
