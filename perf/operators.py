"""The 8-bit operators of a decoder layer's projections, as cases that can be timed and checked.

A case is one call of one operator, as a forward pass makes it:

  quant   rows of an attention's output (or of a weight) to 8 bits with scales
          (specdec.ops.quantize_fp8)
  norm    residual addition, RMS norm and the 8-bit rows that the next
          projection reads (specdec.ops.add_rmsnorm_fp8)
  silu    the MLP's SiLU(gate) * up, written in 8 bits (specdec.ops.silu_mul_fp8)
  linear  a projection: 8-bit rows times an 8-bit weight, with a residual added
          or not (specdec.ops.linear_fp8)

The format: a row of K values is cut into groups of 128 (the last may be
shorter).  A group's scale is the least power of two s, 2^-126 at least, with
max |y| <= 448 s over its finite values; its codes are y / s rounded to e4m3,
infinities and NaN to NaN.  Codes are padded with zeros to whole groups, scales
with ones to a multiple of four.

Sizes are the SmolLM2-1.7B target's and the SmolLM2-135M draft's projections,
one request's verify (k = 4), batches of 8 and 32, and prompts.
"""
import math
import sys
from pathlib import Path

import torch

own = False

GROUP = 128
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one request's verify: five rows of attention output on their way to o_proj
        {"name": "quant_5x2048", "kind": "quant", "rows": 5, "dim": 2048, "dtype": "bf16"},
        # a weight on its way to 8 bits, from a checkpoint in fp32: the target's down projection
        {"name": "quant_2048x8192_f32", "kind": "quant", "rows": 2048, "dim": 8192, "dtype": "f32"},
        # a single new token of the target: latency counts
        {"name": "norm_1x2048", "kind": "norm", "rows": 1, "dim": 2048, "dtype": "bf16", "delta": True},
        # a batch's draft step, whose width ends in half a group
        {"name": "norm_32x576_f32", "kind": "norm", "rows": 32, "dim": 576, "dtype": "f32", "delta": False},
        # four prompts of 1024 tokens entering the target
        {"name": "norm_4096x2048", "kind": "norm", "rows": 4096, "dim": 2048, "dtype": "bf16", "delta": True},
        # a verify of 8 rows, k = 4
        {"name": "silu_40x8192", "kind": "silu", "rows": 40, "dim": 8192, "dtype": "bf16"},
        # the prompts' MLP, a ragged number of tokens
        {"name": "silu_3001x8192", "kind": "silu", "rows": 3001, "dim": 8192, "dtype": "bf16"},
        # the draft's q/k/v projection of one token: the smallest product
        {"name": "linear_1x576x960", "kind": "linear", "rows": 1, "k": 576, "n": 960, "add": False},
        # one request's verify through the target's gate/up
        {"name": "linear_5x2048x16384", "kind": "linear", "rows": 5, "k": 2048, "n": 16384, "add": False},
        # a verify of 8 rows through the target's down projection, into the residual stream
        {"name": "linear_40x8192x2048", "kind": "linear", "rows": 40, "k": 8192, "n": 2048, "add": True},
        # a verify of 32 rows, k = 8, through the target's q/k/v projection
        {"name": "linear_288x2048x6144", "kind": "linear", "rows": 288, "k": 2048, "n": 6144, "add": False},
        # four prompts of 1024 tokens through gate/up
        {"name": "linear_4096x2048x16384", "kind": "linear", "rows": 4096, "k": 2048, "n": 16384, "add": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["quant", "norm", "silu", "linear", "linear", "linear"])
    if kind != "linear":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        # half the widths are the models', half any at all
        dim = rng.choice([576, 1536, 2048, 8192, _log(rng, 40, 8192), _log(rng, 40, 8192), _log(rng, 40, 8192),
                          _log(rng, 40, 8192)])
        case = {"kind": kind, "rows": _log(rng, 1, min(8192, (1 << 24) // dim)), "dim": dim, "dtype": dtype}
        if kind == "norm":
            case["delta"] = rng.random() < 0.7
        return case
    k = rng.choice([576, 1536, 2048, 8192, _log(rng, 64, 8192), _log(rng, 64, 8192)])
    n = rng.choice([576, 960, 2048, 6144, 16384, _log(rng, 64, 16384), _log(rng, 64, 16384), _log(rng, 64, 16384)])
    return {"kind": kind, "rows": _log(rng, 1, min(4096, (1 << 36) // (k * n))), "k": k, "n": n,
            "add": rng.random() < 0.4}


# ------------------------------------------------------------------ inputs --
def _randn(seed, salt, *shape):
    gen = torch.Generator(device="cuda").manual_seed((seed * 7919 + salt) % (1 << 62))
    return torch.randn(*shape, generator=gen, device="cuda")


def _stream(seed, salt, rows, dim, spread=1.0):
    """Activations as a residual stream has them: some features far wider than the rest."""
    wide = torch.exp(0.8 * _randn(seed, salt + 1, dim))
    return spread * wide * _randn(seed, salt, rows, dim)


def _tiled(codes):
    """A weight's codes [N, Kp] in the order in which a wave loads them: blocks
    of 16 features and 128 inputs, 2 KB each, [N / 16, Kp / 128, half, lane, 16],
    lane 16 g + c of half h holding feature c's bytes 64 h + 16 g .. + 15.  Rows
    past N are zeros."""
    n, kp = codes.shape
    rows = -(-n // 16) * 16
    raw = torch.zeros(rows, kp, dtype=torch.uint8, device=codes.device)
    raw[:n] = codes.view(torch.uint8)
    t = raw.view(rows // 16, 16, kp // 128, 2, 4, 16).permute(0, 2, 3, 4, 1, 5)
    return t.reshape(rows // 16, kp // 128, 2, 64, 16).contiguous().view(codes.dtype)


def prepare(case, seed):
    state = dict(case)
    kind = case["kind"]
    if kind == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        x = _stream(seed, 10, rows, k)
        w = 0.02 * _randn(seed, 20, n, k)
        state["x"], state["x_scales"] = _quantized(x)
        # the weight in 8 bits, and laid out once as a model keeps it
        state["w"], state["w_scales"] = _quantized(w)
        state["w_tiled"] = _tiled(state["w"])
        state["residual"] = _stream(seed, 30, rows, n).to(torch.bfloat16) if case["add"] else None
        return state
    dtype = DTYPES[case["dtype"]]
    rows, dim = case["rows"], case["dim"]
    if kind == "silu":
        state["x"] = torch.cat([2 * _randn(seed, 40, rows, dim), _stream(seed, 42, rows, dim)], dim=1).to(dtype)
    else:
        state["x"] = _stream(seed, 50, rows, dim, 2.0).to(dtype)
    if kind == "norm":
        state["delta"] = _stream(seed, 60, rows, dim, 0.5).to(dtype) if case["delta"] else None
        state["weight"] = (1 + 0.2 * _randn(seed, 70, dim)).to(dtype)
    return state


# -------------------------------------------------------------- plain form --
def _quantized(y):
    """y [rows, K] fp32 -> codes e4m3 [rows, Kp], scales e8m0 [rows, Gp]."""
    rows, k = y.shape
    groups = -(-k // GROUP)
    kp, gp = groups * GROUP, -(-k // (4 * GROUP)) * 4
    padded = torch.zeros(rows, kp, dtype=torch.float32, device=y.device)
    padded[:, :k] = y
    padded = padded.view(rows, groups, GROUP)
    finite = torch.isfinite(padded)
    amax = torch.where(finite, padded, torch.zeros_like(padded)).abs().amax(-1)
    # amax = m 2^e with m in [1/2, 1), 448 = 7/8 2^9: the least power of two not
    # below amax / 448
    m, e = torch.frexp(amax)
    e = torch.clamp(torch.where(m > 0.875, e - 8, e - 9), min=-126)
    e = torch.where(amax > 0, e, torch.full_like(e, -126))
    scaled = torch.ldexp(padded, -e.unsqueeze(-1))
    scaled = torch.where(finite, scaled, torch.full_like(scaled, math.nan))
    codes = scaled.to(torch.float8_e4m3fn).view(rows, kp)
    scales = torch.full((rows, gp), 127, dtype=torch.uint8, device=y.device)
    scales[:, :groups] = (e + 127).to(torch.uint8)
    return codes, scales.view(torch.float8_e8m0fnu)


def _values(codes, scales):
    """fp32 values of codes [rows, Kp] and scales [rows, Gp]."""
    rows, kp = codes.shape
    c = codes.to(torch.float32).view(rows, kp // GROUP, GROUP)
    return (c * scales[:, :kp // GROUP].to(torch.float32).unsqueeze(-1)).view(rows, kp)


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "quant":
        return _quantized(state["x"].float())
    if kind == "silu":
        x = state["x"].float()
        gate, up = x[:, :state["dim"]], x[:, state["dim"]:]
        return _quantized(gate / (1 + torch.exp(-gate)) * up)
    if kind == "norm":
        h = state["x"]
        if state["delta"] is not None:
            h = (h.float() + state["delta"].float()).to(h.dtype)
        f = h.float()
        y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * state["weight"].float()
        return (h, *_quantized(y)) if state["delta"] is not None else _quantized(y)
    y = _values(state["x"], state["x_scales"]) @ _values(state["w"], state["w_scales"]).t()
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(torch.bfloat16)


def work(case):
    kind = case["kind"]
    if kind == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        packed = k + -(-k // GROUP)
        return {"bytes": (rows + n) * packed + rows * n * (4 if case["add"] else 2), "flops": 2 * rows * n * k}
    rows, dim = case["rows"], case["dim"]
    size = 2 if case["dtype"] == "bf16" else 4
    packed = dim + -(-dim // GROUP)
    if kind == "quant":
        return {"bytes": rows * (dim * size + packed), "flops": 2 * rows * dim}
    if kind == "silu":
        return {"bytes": rows * (2 * dim * size + packed), "flops": 7 * rows * dim}
    streams = 3 if case["delta"] else 1
    return {"bytes": rows * (streams * dim * size + packed) + dim * size, "flops": 7 * rows * dim}


# --------------------------------------------------------------- 64 bits ----
def _exact_rows(y):
    """The format's codes and scales of y [rows, K] in fp64, by logarithms: each
    group's exponent from log2 and put right by comparison."""
    rows, k = y.shape
    out, scales = [], []
    for lo in range(0, k, GROUP):
        part = y[:, lo:lo + GROUP]
        big = part.abs().masked_fill(~part.isfinite(), 0).max(dim=1, keepdim=True).values
        e = torch.ceil(torch.log2(big.clamp_min(2.0 ** -140) / 448))
        e = torch.where(big > 448 * torch.exp2(e), e + 1, e)
        e = torch.where(big <= 448 * torch.exp2(e - 1), e - 1, e).clamp_min(-126)
        v = part * torch.exp2(-e)
        # e4m3: steps of 2^(exponent - 3), of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        out.append(torch.round(v / step) * step)
        scales.append(torch.exp2(e))
        if part.shape[1] < GROUP:
            out.append(torch.zeros(rows, GROUP - part.shape[1], dtype=y.dtype, device=y.device))
    while len(scales) % 4:
        scales.append(torch.ones(rows, 1, dtype=y.dtype, device=y.device))
    return torch.cat(out, 1), torch.cat(scales, 1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "linear":
        def wide(codes, scales):
            return codes.double() * scales.double().repeat_interleave(GROUP, dim=1)[:, :codes.shape[1]]
        y = torch.mm(wide(s["x"], s["x_scales"]), wide(s["w"], s["w_scales"]).t())
        return y if s["residual"] is None else y + s["residual"].double()
    x = s["x"].double()
    if kind == "quant":
        return _exact_rows(x)
    if kind == "silu":
        gate, up = x.split(case["dim"], dim=1)
        return _exact_rows(gate * up / (torch.exp(-gate) + 1))
    if s["delta"] is None:
        return _exact_rows(s["weight"].double() * x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / case["dim"] + EPS))
    # the norm is that of the stream as it is stored, so its sum is rounded first
    summed = x + s["delta"].double()
    stored = summed.to(s["x"].dtype).double()
    y = s["weight"].double() * stored / torch.sqrt(stored.pow(2).sum(1, keepdim=True) / case["dim"] + EPS)
    return (summed, *_exact_rows(y))


# ------------------------------------------------------ the framework's own --
def _run_own(state):
    package = str(Path(__file__).resolve().parent.parent / "speculative-decoder_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from specdec import ops

    kind = state["kind"]
    if kind == "quant":
        return ops.quantize_fp8(state["x"])
    if kind == "silu":
        return ops.silu_mul_fp8(state["x"])
    if kind == "norm":
        if state["delta"] is None:
            return ops.add_rmsnorm_fp8(state["x"], None, state["weight"], EPS)
        summed = torch.empty_like(state["x"])
        return (summed, *ops.add_rmsnorm_fp8(state["x"], state["delta"], state["weight"], EPS, summed=summed))
    return ops.linear_fp8(state["x"], state["x_scales"], state["w_tiled"], state["w_scales"], add=state["residual"])
