"""Rates at which the pairs of a head turn with the position, for `ck.paged_write_rope`."""
from __future__ import annotations

import math

import torch


def rope_rates(dim: int, base: float = 10000.0, factor: float = 1.0, context: int = 0, slow: float = 1.0, fast: float = 32.0,
               device: torch.device | str = "cuda") -> torch.Tensor:
    """base ** (-2i / dim) for i < dim / 2, fp32 on the device; dim: the elements of a head that turn, even.

    factor > 1 makes room for contexts `factor` times as long as those a model was trained on.  With context 0
    every rate is divided by it.  With the trained context, only the slow pairs' are: those that turn less
    than `slow` times over it wholly, those that turn over `fast` times not at all, those between by the share
    that lies between, (turns - slow) / (fast - slow) of a pair's own rate and the rest of the divided one.
    Checkpoints that were trained with another ramp, such as one that is linear in a pair's number between two
    pairs, need rates of their own: `ck.paged_write_rope` takes any.
    """
    if dim < 0 or dim % 2:
        raise ValueError(f"rope_rates: {dim} elements do not make pairs")
    if not (base > 0 and factor > 0 and context >= 0 and (context == 0 or fast > slow)):
        raise ValueError(f"rope_rates: base {base}, factor {factor}, context {context}, slow {slow}, fast {fast}")
    rates = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim) if dim else torch.empty(0, dtype=torch.float64)
    own = ((context * rates / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1) if context else torch.zeros_like(rates)
    return (rates * (own + (1 - own) / factor)).float().to(device)
