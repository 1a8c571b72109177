"""The tree operators together: verification of drafted trees, the round loop
and its drafter, on tiny models and on the target's layer shapes."""
import pytest
import torch

from baselines import cached_autoregressive
from cache.kv import KVCache
from lm.forward import forward, forward_core
from lm.model import SMOLLM2_135M, SMOLLM2_1_7B, Llama, as_llama
from lm.sampling import draw, filtered_probabilities
from lm.tree import TreeStep, plan
from spec.tree import ModelTree, generate_tree, tree_shape, verify_tree
from tiny_models import early_exit, random_prompts, tiny64
from tree_ref import ancestors
import tree_ref

pytestmark = pytest.mark.gpu


def cache_for(model, dtype=torch.float32, blocks=128, bs=16):
    return KVCache.for_model(model.config, blocks, bs, dtype, "cuda")


def path_logits(model, prompt, tokens, parents, dtype=torch.float32):
    """The logits after each node, each from a plain forward over the prompt and the node's path."""
    seen, _ = ancestors(parents)
    out = []
    for i in range(tokens.shape[1]):
        chain = tokens[0, seen[0, i]].tolist()
        cache = cache_for(model, dtype)
        cache.add(0)
        ids = torch.tensor([prompt[:-1] + chain])
        out.append(forward(model, cache, [0], ids, [ids.shape[1]])[0, -1])
    return torch.stack(out)


@pytest.mark.parametrize("dtype,off", [(torch.float32, 2e-4), (torch.bfloat16, 0.15)])
def test_tree_forward_equals_a_forward_of_each_path(dtype, off):
    """fp32: two orders of sums through two layers.  bf16: some ten roundings of
    2^-8 on the way through each, of logits up to a few units."""
    model = tiny64(3, dtype)
    parents = tree_shape([3, 2, 1])
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, 256, (37,), generator=g).tolist()
    tokens = torch.randint(0, 256, (1, parents.shape[1]), generator=g)
    tokens[0, 0] = prompt[-1]
    cache = cache_for(model, dtype)
    cache.add(0)
    forward(model, cache, [0], torch.tensor([prompt[:-1]]), [len(prompt) - 1])
    llama = as_llama(model, "cuda")
    step = cache.append([0], [4], nodes=[parents.shape[1]])
    mask, depth = (t.cuda() for t in plan(parents))
    tree = TreeStep(mask, depth, TreeStep.store(llama, 1, parents.shape[1]), step.past[0])
    got = forward_core(llama, cache, step.meta, tokens.cuda(), step.past[0], tree=tree)[0]
    want = path_logits(model, prompt, tokens, parents, dtype)
    scale = want.abs().max()
    assert bool(((got - want).abs() <= off * scale).all()), float(((got - want).abs() / scale).max())


def test_verify_then_plain_forward_reads_the_committed_path():
    """After the commit a plain forward over the cache gives what a fresh prefill gives."""
    model = tiny64(4)
    parents = tree_shape([2, 2, 1])
    prompt = random_prompts(1, 256, 7, 30, 31)[0]
    # a tree that holds the target's own greedy continuation on one path
    greedy = cached_autoregressive.generate(model, cache_for(model), prompt, 4)
    tokens = torch.randint(0, 256, (1, parents.shape[1]), generator=torch.Generator().manual_seed(1))
    tokens[0, 0] = prompt[-1]
    for node, token in zip((2, 5, 9), greedy):  # 0 -> 2 -> 5 -> 9
        tokens[0, node] = token
    assert [int(parents[0, i]) for i in (2, 5, 9)] == [0, 2, 5]
    cache = cache_for(model)
    cache.add(0)
    forward(model, cache, [0], torch.tensor([prompt[:-1]]), [len(prompt) - 1])
    verdict = verify_tree(model, cache, [0], [prompt], tokens, parents, torch.zeros(1, parents.shape[1]))[:, 0].tolist()
    assert verdict[0] == 3 and verdict[2:5] == greedy[:3] and verdict[1] == greedy[3]
    cache.truncate(0, len(prompt) + 3)
    got = forward(model, cache, [0], torch.tensor([[verdict[1]]]), [1])[0, 0]
    fresh = cache_for(model)
    fresh.add(0)
    ids = torch.tensor([prompt + greedy[:4]])
    want = forward(model, fresh, [0], ids, [ids.shape[1]])[0, -1]
    assert bool(((got - want).abs() <= 2e-4 * want.abs().max()).all())


@pytest.mark.parametrize("branching", [[1], [4], [3, 2], [2, 2, 2], [1, 1, 1, 1, 1]])
def test_greedy_trees_equal_plain_greedy(branching):
    target = tiny64(0)
    draft = early_exit(target)
    prompts = random_prompts(4, 256, 11)
    plain = [cached_autoregressive.generate(target, cache_for(target), p, 24) for p in prompts]
    out, stats = generate_tree(target, cache_for(target), ModelTree(draft, cache_for(draft), branching), prompts, 24)
    assert out == plain
    assert 0 < stats.accepted <= stats.drafted and sum(stats.emitted_per_round) == 4 * 23


def test_the_target_as_its_own_draft_accepts_every_level():
    target = tiny64(0)
    prompts = random_prompts(3, 256, 12)
    out, stats = generate_tree(target, cache_for(target), ModelTree(target, cache_for(target), [2, 1, 1]), prompts, 17)
    plain = [cached_autoregressive.generate(target, cache_for(target), p, 17) for p in prompts]
    assert out == plain and stats.rounds == 4  # 1 + 4 x 4 tokens


def test_eos_and_budget_end_rows_apart():
    target = tiny64(0)
    prompts = random_prompts(5, 256, 13)
    plain = [cached_autoregressive.generate(target, cache_for(target), p, 30) for p in prompts]
    eos = plain[0][9]
    want = [p[:p.index(eos) + 1] if eos in p else p for p in plain]
    cache, draft_cache = cache_for(target), cache_for(target)
    out, _ = generate_tree(target, cache, ModelTree(early_exit(target), cache_for(early_exit(target)), [2, 2]), prompts, 30,
                           eos_id=eos)
    assert out == want
    assert cache.allocator.num_used == 0


def test_sampled_trees_draw_what_plain_sampling_draws():
    """With one branch the uniforms of a chain's nodes are those of its tokens: the
    emitted tokens are draws from the target's restricted distribution at their own
    contexts, whatever the draft proposed."""
    target = tiny64(2)
    prompts = random_prompts(2, 256, 14)
    kw = dict(temperature=0.9, top_k=20, top_p=0.95, min_p=0.01)
    drafter = ModelTree(early_exit(target), cache_for(early_exit(target)), [2, 1])
    gen = torch.Generator().manual_seed(3)
    replay = torch.Generator().manual_seed(3)
    out, stats = generate_tree(target, cache_for(target), drafter, prompts, 12, generator=gen, **kw)
    for p, o in zip(prompts, out):
        assert len(o) == 12
        # each token is among those that its context's distribution keeps
        cache = cache_for(target)
        cache.add(0)
        ids = torch.tensor([p + o])
        logits = forward(target, cache, [0], ids, [ids.shape[1]])[0, len(p) - 1:-1]
        probs = filtered_probabilities(logits, **kw).cpu()
        assert bool((probs[torch.arange(12), torch.tensor(o)] > 0).all())
    # the first tokens, from the same uniforms
    u = torch.rand(2, generator=replay)
    for p, o, v in zip(prompts, out, u):
        cache = cache_for(target)
        cache.add(0)
        logits = forward(target, cache, [0], torch.tensor([p]), [len(p)])[0, -1]
        assert int(draw(logits, v.view(()), **kw)) == o[0]


def test_filtered_probabilities_and_draws_agree_with_a_sort():
    logits = 3 * torch.randn(5, 400, generator=torch.Generator().manual_seed(1))
    probs = filtered_probabilities(logits, 0.8, 30, 0.9, 0.02).cpu()
    u = torch.rand(5, generator=torch.Generator().manual_seed(2))
    got = draw(logits, u, 0.8, 30, 0.9, 0.02).cpu()
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
    for r in range(5):
        token, want, _ = tree_ref.draw(logits[r], float(u[r]), f32(0.8), 30, f32(0.9), f32(0.02))
        assert int(got[r]) == token and torch.allclose(probs[r].double(), want, rtol=2.0 ** -22, atol=0)


@pytest.mark.parametrize("eight", [False, True])
def test_the_models_shapes(eight):
    """The target's and the draft's layer shapes in bf16 (and 8 bits): rows of
    different lengths through a whole round loop; caches come back empty."""
    ts, ds = SMOLLM2_1_7B.replace(num_hidden_layers=2), SMOLLM2_135M.replace(num_hidden_layers=2)
    target, draft = Llama.random(ts, 0, "cuda"), Llama.random(ds, 1, "cuda")
    if eight:
        target = target.fp8()
    tc, dc = (KVCache.for_model(s, 128, 16, torch.bfloat16, "cuda") for s in (ts, ds))
    prompts = random_prompts(3, 49152, 15, 20, 90)
    out, stats = generate_tree(target, tc, ModelTree(draft, dc, [4, 2, 1]), prompts, 10, temperature=0.8, top_p=0.9)
    assert [len(o) for o in out] == [10] * 3 and stats.drafted > 0
    assert tc.allocator.num_used == 0 and dc.allocator.num_used == 0


def test_a_wide_tree_of_several_mask_words():
    target = tiny64(0)
    prompts = random_prompts(2, 256, 16)
    plain = [cached_autoregressive.generate(target, cache_for(target), p, 9) for p in prompts]
    drafter = ModelTree(early_exit(target), cache_for(early_exit(target)), [5, 4, 3, 1])  # 146 nodes
    out, _ = generate_tree(target, cache_for(target), drafter, prompts, 9)
    assert out == plain
