"""The table of cosines and sines that ``ops.rope`` and the indexer prologue read, on MI355X.

Pair p of a rotated head of ``rot_dim`` turns by position * f_p, f_p = base^(-2p / rot_dim). For contexts ``factor``
times as long as the model was trained on (``original_max_position``), YaRN (Peng et al., 2023) keeps the pairs that turn
beta_fast times or more over the original context, slows those of fewer than beta_slow turns by ``factor``, and blends
in between:

    pair(r) = rot_dim ln(original_max_position / (2 pi r)) / (2 ln base)   (the pair that turns r times)
    low, high = floor(pair(beta_fast)), ceil(pair(beta_slow)), both from 0 to rot_dim - 1
    keep_p  = 1 - clamp((p - low) / (high - low), 0, 1)
    f_p     = base^(-2p / rot_dim) (keep_p + (1 - keep_p) / factor)

with cosines and sines times ``attention_factor`` (0.1 ln(factor) + 1 unless given; 1 where the attention's scale
carries it). Angles and their cosines are taken in float64 and rounded once: a position of 2^20 in float32 would leave
its angle with an error of 2^-4.
"""
from __future__ import annotations

import math

import torch


def inverse_frequencies(rot_dim: int, base: float = 10000.0, *, factor: float = 1.0,
                        original_max_position: int | None = None, beta_fast: float = 32.0,
                        beta_slow: float = 1.0) -> torch.Tensor:
    """f_p of the rot_dim / 2 pairs, float64 on the CPU."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be even and positive, got {rot_dim}")
    if not (base > 1 and factor >= 1 and beta_fast > beta_slow > 0):
        raise ValueError(f"base > 1, factor >= 1 and beta_fast > beta_slow > 0 are needed, got {base}, {factor}, "
                         f"{beta_fast}, {beta_slow}")
    pairs = torch.arange(rot_dim // 2, dtype=torch.float64)
    freq = torch.pow(torch.tensor(base, dtype=torch.float64), -2.0 * pairs / rot_dim)
    if factor == 1:
        return freq
    if original_max_position is None or original_max_position < 1:
        raise ValueError("a factor needs the original_max_position that it extends")

    def pair(turns: float) -> float:
        return rot_dim * math.log(original_max_position / (2 * math.pi * turns)) / (2 * math.log(base))

    low = max(math.floor(pair(beta_fast)), 0)
    high = min(math.ceil(pair(beta_slow)), rot_dim - 1)
    keep = 1 - ((pairs - low) / max(high - low, 1e-3)).clamp(0, 1)
    return freq * (keep + (1 - keep) / factor)


def cos_sin_cache(max_position: int, rot_dim: int, base: float = 10000.0, *, factor: float = 1.0,
                  original_max_position: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                  attention_factor: float | None = None, device="cuda") -> torch.Tensor:
    """[max_position, rot_dim] float32 = [cos | sin] of each position's angles, the table of ``ops.rope`` and, for
    rot_dim 64, of the indexer prologue."""
    if max_position < 1:
        raise ValueError(f"max_position must be positive, got {max_position}")
    freq = inverse_frequencies(rot_dim, base, factor=factor, original_max_position=original_max_position,
                               beta_fast=beta_fast, beta_slow=beta_slow)
    if attention_factor is None:
        attention_factor = 0.1 * math.log(factor) + 1.0
    out = torch.empty(max_position, rot_dim, dtype=torch.float32, device=device)
    step = 1 << 16  # (float64 angles of so many positions at a time)
    for at in range(0, max_position, step):
        angle = torch.outer(torch.arange(at, min(at + step, max_position), dtype=torch.float64), freq)
        out[at:at + step] = (torch.cat([angle.cos(), angle.sin()], dim=1) * attention_factor).float()
    return out
