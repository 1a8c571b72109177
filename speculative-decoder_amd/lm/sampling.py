"""Temperature sampling helpers (reference: lm/sampling.py:4-18).

`probabilities` runs the softmax / one-hot kernel of libspecdec.so.
"""
from __future__ import annotations

import torch

from specdec import ops


def next_token(logits: torch.Tensor, temperature: float, generator: torch.Generator | None) -> int:
    """logits: [V].  Temperature 0 is greedy (the first maximum wins, so ties go
    to the lower id); otherwise one multinomial draw from the softmax with
    `generator` (on the generator's device)."""
    if temperature == 0.0:
        return int(torch.argmax(logits))
    probs = probabilities(logits, temperature)
    dev = generator.device if generator is not None else torch.device("cpu")
    return int(torch.multinomial(probs.to(dev), 1, generator=generator))


def draw(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """A token id for each row of logits [..., V] from the row's uniform u [...]
    (fp32), under temperature, top-k, top-p and min-p (numbers, or tensors of a
    value a row): `ops.sample`, for logits and uniforms wherever they are."""
    if logits.device.type != "cuda":
        logits = logits.to("cuda")
    return ops.sample(logits, u.to(logits.device, non_blocking=True), temperature, top_k, top_p, min_p)


def filtered_probabilities(logits: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """`probabilities` restricted to what top-k, top-p and min-p keep of each row
    of logits [..., V], fp32, renormalised: accept-reject between a target's and
    a draft's emits the target's restricted distribution."""
    if logits.device.type != "cuda":
        logits = logits.to("cuda")
    probs = torch.empty(logits.shape, dtype=torch.float32, device=logits.device)
    ops.sample(logits, torch.zeros(logits.shape[:-1], device=logits.device), temperature, top_k, top_p, min_p, probs=probs)
    return probs


def probabilities(logits: torch.Tensor, temperature: float) -> torch.Tensor:
    """[..., V] logits -> float32 probabilities on the logits' GPU.  Temperature
    0 gives the one-hot of the argmax (lowest id among ties), which turns
    accept-reject into exact greedy verification."""
    if logits.device.type != "cuda":
        logits = logits.to("cuda")
    return ops.probabilities(logits, temperature)
