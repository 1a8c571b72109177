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


def plain_logits(model, context):
    """The logits after a context, by a forward over all of it."""
    cache = cache_for(model)
    cache.add(0)
    return forward(model, cache, [0], torch.tensor([context]), [len(context)])[0, -1].float().cpu()


@pytest.mark.parametrize("branching", [[2], [3, 2, 1], [1, 1, 1]])
def test_each_token_is_drawn_with_its_node_s_uniform(branching):
    """The generator replayed: the first tokens', then for each round a uniform a row
    and node.  From node 0 the token is the draw from the target's restricted
    distribution after the path, by a plain forward and a sort in 64 bits, with the
    uniform of the path's node; where a child carries it the path goes on there.  The
    tree's sums are ordered otherwise than a plain forward's (2e-4 of the logits), so
    a u nearer to its token's border than 1e-3 of the mass tells nothing.  The same
    with another node's uniforms has to disagree."""
    target = tiny64(2)
    prompts = random_prompts(3, 256, 14)
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
    kw = dict(temperature=0.9, top_k=20, top_p=0.95, min_p=0.01)
    drafter = ModelTree(early_exit(target), cache_for(early_exit(target)), branching)
    proposals = []
    propose = drafter.propose

    def recorded(seq_ids, contexts):
        tokens, parents = propose(seq_ids, contexts)
        proposals.append((list(seq_ids), [list(c) for c in contexts], tokens.cpu(), parents))
        return tokens, parents

    drafter.propose = recorded
    out, stats = generate_tree(target, cache_for(target), drafter, prompts, 14,
                               generator=torch.Generator().manual_seed(3), **kw)
    final = [p + o for p, o in zip(prompts, out)]
    assert stats.accepted > 0 and [len(o) for o in out] == [14] * 3

    def drawn(context, u):
        token, _, gap = tree_ref.draw(plain_logits(target, context), float(u), f32(0.9), 20, f32(0.95), f32(0.01))
        return token, gap

    replay = torch.Generator().manual_seed(3)
    for p, f, u in zip(prompts, final, torch.rand(3, generator=replay)):
        token, gap = drawn(p, u)
        assert f[len(p)] == token or gap < 1e-3
    told, other, deep = 0, 0, 0
    for ids, contexts, tokens, parents in proposals:
        u = torch.rand(*tokens.shape, generator=replay)
        for row, (seq, context) in enumerate(zip(ids, contexts)):
            node, at = 0, len(context)
            assert context == final[seq][:at]
            while at < len(final[seq]):
                token, gap = drawn(final[seq][:at], u[row, node])
                assert final[seq][at] == token or gap < 1e-3, (seq, at, node)
                told += gap >= 1e-3
                deep += node > 0
                wrong, wrong_gap = drawn(final[seq][:at], u[row, (node + 1) % u.shape[1]])
                other += wrong != final[seq][at] and wrong_gap >= 1e-3
                token, at = final[seq][at], at + 1
                child = [c for c in range(node + 1, tokens.shape[1])
                         if int(parents[0, c]) == node and int(tokens[row, c]) == token]
                if not child:
                    break
                node = child[0]
    assert told > 20 and deep > 0 and other > 0


def test_a_verify_that_fails_leaves_the_cache_as_it_was():
    """A tree of too many nodes, uniforms, rows or parents of another size, a
    parameter out of range and too few blocks: the rows' lengths and blocks stay, and
    a right call after them works."""
    model = tiny64(1)
    prompts = random_prompts(2, 256, 18)
    cache = cache_for(model, blocks=8)
    for s, p in enumerate(prompts):
        cache.add(s)
        forward(model, cache, [s], torch.tensor([p[:-1]]), [len(p) - 1])
    lengths, used = [cache.length(s) for s in (0, 1)], cache.allocator.num_used
    parents = tree_shape([2, 1])
    tokens = torch.randint(0, 256, (2, 5), generator=torch.Generator().manual_seed(0))
    tokens[:, 0] = torch.tensor([p[-1] for p in prompts])
    u = torch.rand(2, 5, generator=torch.Generator().manual_seed(1))
    good = dict(target=model, cache=cache, seq_ids=[0, 1], contexts=prompts, tokens=tokens, parents=parents, u=u)
    wide, chain = tree_shape([255]), tree_shape([1] * 200)
    for kind, change in [
            (ValueError, dict(tokens=torch.zeros(2, 257, dtype=torch.int64), parents=torch.cat([wide, wide[:, -1:]], 1), u=torch.rand(2, 257))),
            (ValueError, dict(u=u[:, :4])), (ValueError, dict(u=u[:1])), (ValueError, dict(tokens=tokens[:1])),
            (ValueError, dict(tokens=tokens[0])), (ValueError, dict(parents=parents[:, :4])), (ValueError, dict(parents=parents[0])),
            (ValueError, dict(parents=parents.repeat(3, 1))), (ValueError, dict(top_p=1.5)), (ValueError, dict(temperature=-1.0)),
            (Exception, dict(tokens=torch.zeros(2, 201, dtype=torch.int64), parents=chain, u=torch.rand(2, 201)))]:
        with pytest.raises(kind):
            verify_tree(**{**good, **change})
        assert [cache.length(s) for s in (0, 1)] == lengths, change.keys()
        assert cache.allocator.num_used == used, change.keys()
    verdict = verify_tree(**good)
    for b, p in enumerate(prompts):
        alone = cache_for(model)
        alone.add(0)
        forward(model, alone, [0], torch.tensor([p[:-1]]), [len(p) - 1])
        one = verify_tree(model, alone, [0], [p], tokens[b:b + 1], parents, u[b:b + 1])
        assert verdict[:, b].tolist() == one[:, 0].tolist()
