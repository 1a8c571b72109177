"""The bytes of weights that the bench charges a forward with, as stored."""
import torch

import bench
from lm.model import Fp8Layer, Llama, LlamaShape
from specdec import ops

SHAPE = LlamaShape(vocab_size=96, hidden_size=128, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1,
                   intermediate_size=200)
# q/k/v, o, gate/up and down: features, inputs
PROJECTIONS = [(256, 128), (128, 128), (400, 128), (128, 200)]


def head_bytes(llama):
    return llama.head_wide.numel() * llama.head_wide.element_size()


def test_weights_in_the_models_type():
    llama = Llama.random(SHAPE, 0, "cpu")
    assert bench.weight_bytes(llama) == 2 * sum(2 * n * k for n, k in PROJECTIONS) + head_bytes(llama)


def test_weights_in_8_bits():
    """Codes padded to whole tiles of 16 features x 128 inputs, and a scale byte for each 128, four at least."""
    def weight(n, k):
        codes = torch.zeros(n, -(-k // 128) * 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
        return ops.tile_weight_fp8(codes), torch.zeros(n, -(-k // 512) * 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)

    llama = Llama.random(SHAPE, 0, "cpu")
    llama.layers = [Fp8Layer(*(weight(n, k) for n, k in PROJECTIONS)) for _ in range(2)]
    assert llama.is_fp8
    a_layer = sum(-(-n // 16) * 16 * -(-k // 128) * 128 + n * -(-k // 512) * 4 for n, k in PROJECTIONS)
    assert bench.weight_bytes(llama) == 2 * a_layer + head_bytes(llama)
