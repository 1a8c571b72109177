"""A model with 8-bit projections (Llama.fp8) through the forward, the round
loop and plain decoding."""
import pytest
import torch

from baselines import cached_autoregressive
from cache.kv import KVCache
from lm.forward import forward
from lm.model import SMOLLM2_135M, SMOLLM2_1_7B, Fp8Layer, Llama, LlamaShape, rope_tables
from spec.draft import ModelDraft
from spec.loop import generate
from spec.ngram import NGramDraft
from test_gpu_fp8 import ref_codes, ref_scale_exponents

pytestmark = pytest.mark.gpu
G = 128


def in_8_bits(y):
    """The values that rows y [R, K] (fp64) stand for in the 8-bit format."""
    e, _ = ref_scale_exponents(y)
    q = ref_codes(y, e) * torch.exp2(e.double()).repeat_interleave(G, dim=1)
    return q[:, :y.shape[1]]


def plain_logits(llama, ids):
    """The model in fp64 from the operators' definitions: weights and the rows
    before each projection in the 8-bit format, all else unrounded.  ids [T]."""
    cfg = llama.config
    h, hk, d = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    t = len(ids)
    x = llama.embed.cpu().double()[ids]
    cos, sin = (v[:t].double() for v in rope_tables(cfg, t))

    def norm(v):
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + cfg.rms_norm_eps)

    def rot(v):  # [T, heads, d]
        a, b = v[..., : d // 2], v[..., d // 2:]
        c, s = cos[:, None], sin[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    def project(rows, w):
        return in_8_bits(rows) @ in_8_bits(w.cpu().double()).t()

    for layer in llama.layers:
        qkv = project(norm(x), layer.wqkv)
        q, k, v = qkv.split([h * d, hk * d, hk * d], dim=1)
        q, k, v = rot(q.view(t, h, d)), rot(k.view(t, hk, d)), v.view(t, hk, d)
        k, v = k.repeat_interleave(h // hk, 1), v.repeat_interleave(h // hk, 1)
        scores = torch.einsum("qhd,khd->hqk", q, k) * llama.scaling
        scores = scores.masked_fill(torch.ones(t, t).triu(1).bool(), float("-inf"))
        attn = torch.einsum("hqk,khd->qhd", scores.softmax(-1), v).reshape(t, h * d)
        x = x + project(attn, layer.wo)
        gate, up = project(norm(x), layer.wgu).chunk(2, dim=1)
        x = x + project(gate / (1 + torch.exp(-gate)) * up, layer.wd)
    return (norm(x) * llama.norm.cpu().double()) @ llama.head_wide.cpu().double().t()


# widths that end inside a group (320, 832), five query heads to a kv head
ODD = LlamaShape(vocab_size=512, hidden_size=320, num_hidden_layers=2, num_attention_heads=5, num_key_value_heads=1,
                 intermediate_size=832)


@pytest.mark.parametrize("length", [1, 5, 40, 150])
def test_forward_matches_the_definition(length):
    """Against the definition the kernels round each bf16 tensor between the
    operators (2^-9 rms at most, about ten of them in a layer: 1%), and codes of
    values so near a border flip (a code's step is 2^-3 of its value: a bf16
    step moves one value in 32 over a border, sqrt(1 / 32) * 2^-4 = 1% a
    projection, eight of them).  A wrong scale, group or weight is off by 1."""
    llama = Llama.random(ODD, 3, "cuda")
    ids = torch.randint(0, 512, (length,), generator=torch.Generator().manual_seed(length)).tolist()
    want = plain_logits(llama, ids)
    q8 = llama.fp8()
    assert all(isinstance(layer, Fp8Layer) for layer in q8.layers) and q8.fp8() is q8
    cache = KVCache.for_model(ODD, 32, 16, torch.bfloat16, "cuda")
    cache.add(0)
    got = forward(q8, cache, [0], torch.tensor([ids]), [length])[0].cpu().double()
    assert ((got - want).norm() / want.norm()).item() < 0.05
    # and it is a rounding of the bf16 model
    cache.add(1)
    base = forward(llama, cache, [1], torch.tensor([ids]), [length])[0].cpu().double()
    assert ((got - base).norm() / base.norm()).item() < 0.25


def test_padded_batches_match_single_rows():
    """A right-padded batch of few rows: each sequence has the bits of its own call."""
    q8 = Llama.random(ODD, 5, "cuda").fp8()
    g = torch.Generator().manual_seed(6)
    rows = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (3, 12, 1, 7)]
    width = max(map(len, rows))
    cache = KVCache.for_model(ODD, 64, 16, torch.bfloat16, "cuda")
    for s in range(8):
        cache.add(s)
    ids = torch.tensor([r + [0] * (width - len(r)) for r in rows])
    together = forward(q8, cache, [0, 1, 2, 3], ids, [len(r) for r in rows])
    for i, r in enumerate(rows):
        alone = forward(q8, cache, [4 + i], torch.tensor([r]), [len(r)])
        assert torch.equal(alone[0], together[i, :len(r)]), i


@pytest.mark.parametrize("drafter", ["model", "ngram"])
def test_speculative_output_is_plain_greedy_output(drafter):
    ts, ds = SMOLLM2_1_7B.replace(num_hidden_layers=2), SMOLLM2_135M.replace(num_hidden_layers=2)
    target, draft = Llama.random(ts, 0, "cuda").fp8(), Llama.random(ds, 1, "cuda").fp8()
    g = torch.Generator().manual_seed(31)
    for n in (20, 96):
        prompt = torch.randint(0, 49152, (n,), generator=g).tolist()
        tc = KVCache.for_model(ts, 64, 16, torch.bfloat16, "cuda")
        d = (ModelDraft(draft, KVCache.for_model(ds, 64, 16, torch.bfloat16, "cuda")) if drafter == "model"
             else NGramDraft(49152))
        out, _ = generate(target, tc, d, [prompt], 40, k=4)
        plain = cached_autoregressive.generate(target, KVCache.for_model(ts, 64, 16, torch.bfloat16, "cuda"), prompt, 40)
        assert out[0] == plain


def test_own_draft_is_always_accepted():
    """The 8-bit target as its own draft at temperature 0 with the verify's
    split: every draft is accepted, eager and captured calls in turn."""
    ts = SMOLLM2_135M.replace(num_hidden_layers=3)
    target = Llama.random(ts, 2, "cuda").fp8()
    prompt = torch.randint(0, 49152, (50,), generator=torch.Generator().manual_seed(1)).tolist()
    tc, dc = (KVCache.for_model(ts, 64, 16, torch.bfloat16, "cuda") for _ in range(2))
    out, stats = generate(target, tc, ModelDraft(target, dc, exact=True), [prompt], 30, k=4)
    assert len(out[0]) == 30 and stats.accepts == stats.attempts


def test_fp8_refusals():
    with pytest.raises(NotImplementedError):
        Llama.random(ODD, 3, "cpu").fp8()
    with pytest.raises(NotImplementedError):
        Llama.random(ODD, 3, "cuda", torch.float32).fp8()
