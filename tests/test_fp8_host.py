"""What the 8-bit operators refuse before anything is launched, and the layout
of a tiled weight (no GPU needed)."""
import pytest
import torch

from specdec import _lib, ops

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def test_cpu_inputs_are_refused():
    x = torch.randn(2, 300)
    codes, scales = torch.zeros(2, 384, dtype=torch.uint8).view(F8), torch.full((2, 4), 127, dtype=torch.uint8).view(E8)
    w = torch.zeros(1, 3, 2, 64, 16, dtype=torch.uint8).view(F8)
    for call in (lambda: ops.quantize_fp8(x), lambda: ops.silu_mul_fp8(x),
                 lambda: ops.add_rmsnorm_fp8(x, None, torch.ones(300), 1e-5),
                 lambda: ops.linear_fp8(codes, scales, w, scales)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_tiled_weight_layout():
    """Every element of a tiled weight by the index the C ABI documents, and zeros past N."""
    n, kp = 37, 384
    raw = (torch.arange(n * kp) % 127).to(torch.uint8).reshape(n, kp)
    t = ops.tile_weight_fp8(raw.view(F8))
    assert tuple(t.shape) == (3, 3, 2, 64, 16) and t.is_contiguous()
    flat = t.view(torch.uint8).reshape(-1)
    nn, kk = torch.meshgrid(torch.arange(n), torch.arange(kp), indexing="ij")
    pos = ((nn // 16 * (kp // 128) + kk // 128) * 2048 + (kk % 128 // 64) * 1024 +
           ((kk % 64 // 16) * 16 + nn % 16) * 16 + kk % 16)
    assert torch.equal(flat[pos], raw)
    rest = torch.ones(flat.numel(), dtype=torch.bool)
    rest[pos.reshape(-1)] = False
    assert int(rest.sum()) == 11 * kp and bool((flat[rest] == 0).all())
    for bad in (torch.zeros(4, 100, dtype=torch.uint8).view(F8), torch.zeros(4, 128), raw[:0].view(F8),
                raw[0].view(F8)):
        with pytest.raises(ValueError):
            ops.tile_weight_fp8(bad)


def test_c_entries_check_their_arguments_before_launch():
    lib = _lib.load()
    fake = 1 << 20  # never dereferenced: each call returns before any launch
    bf16, f32, f64 = 2, 0, 1
    q = lib.specdec_quantize_fp8
    assert q(fake, f32, 0, 8, 8, fake, fake, None) == 0  # no rows: nothing to do
    assert q(fake, f32, -1, 8, 8, fake, fake, None) == 1
    assert q(fake, f32, 2, 0, 8, fake, fake, None) == 1
    assert q(fake, f32, 2, 8, 7, fake, fake, None) == 1  # rows that overlap
    assert q(fake, f64, 2, 8, 8, fake, fake, None) == 1
    assert q(None, f32, 2, 8, 8, fake, fake, None) == 1
    assert q(fake, f32, 2, 8, 8, fake + 8, fake, None) == 1  # codes 16-byte aligned
    assert q(fake, f32, 2, 8, 8, fake, fake + 2, None) == 1  # scales 4-byte aligned
    assert q(fake, f32, 1 << 28, 8, 8, fake, fake, None) == 3
    s = lib.specdec_silu_mul_fp8
    assert s(fake, bf16, 2, 8, 15, fake, fake, None) == 1  # a row is gate and up
    assert s(fake, bf16, 2, 8, 16, None, fake, None) == 1
    n = lib.specdec_add_rmsnorm_fp8
    assert n(fake, None, fake, None, bf16, 0, 64, 1e-5, fake, fake, None) == 0
    assert n(fake, fake, fake, None, bf16, 1, 64, 1e-5, fake, fake, None) == 1  # a delta and nowhere to write the sum
    assert n(fake, None, None, None, bf16, 1, 64, 1e-5, fake, fake, None) == 1
    assert n(fake, None, fake, None, bf16, 1, 16385, 1e-5, fake, fake, None) == 3
    m = lib.specdec_linear_fp8

    def mm(x=fake, xst=256, xs=fake, xsst=4, w=fake, ws=fake, rows=2, k=256, nf=48, add=None, addst=0, out=fake,
           outst=48):
        return m(x, xst, xs, xsst, w, ws, rows, k, nf, add, addst, out, outst, None)

    assert mm(rows=0) == 0
    assert mm(rows=-1) == 1 and mm(k=200) == 1 and mm(k=0) == 1 and mm(nf=0) == 1
    assert mm(xst=240) == 1 and mm(xsst=2) == 1 and mm(outst=47) == 1 and mm(add=fake, addst=47) == 1
    assert mm(xst=264) == 1 and mm(x=fake + 8) == 1 and mm(w=fake + 4) == 1 and mm(xs=fake + 1) == 1
    assert mm(x=None) == 1 and mm(out=None) == 1 and mm(ws=None) == 1
    assert mm(rows=1048561) == 3 and mm(nf=1 << 25, outst=1 << 25) == 3
    assert mm(xst=(1 << 25) + 16) == 3 and mm(xsst=(1 << 25) + 4) == 3 and mm(k=1 << 24, xst=1 << 24, xsst=1 << 17) == 3


def test_models_off_the_gpu_or_in_fp32_have_no_8_bit_form():
    from lm.model import Llama, LlamaShape

    shape = LlamaShape(vocab_size=32, hidden_size=64, num_hidden_layers=1, num_attention_heads=1, num_key_value_heads=1,
                       intermediate_size=64)
    with pytest.raises(NotImplementedError):
        Llama.random(shape, 0, "cpu").fp8()
