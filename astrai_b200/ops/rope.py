"""Interleaved rotary position embedding.

Parity: astrai/model/components/rope.py. Angles ``pos * base^(-2i/d)`` are
computed in float64 and stored as fp32 (cos, sin) pairs; pairs (x[2i],
x[2i+1]) are rotated. NTK scaling changes the base to
``base * factor^(d/(d-2))``.

On CUDA the rotation runs in place on the q / k column ranges of the fused
QKV projection output, so q and k are never copied.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from astrai_b200.ops._ext import native


def ntk_base(base: float, dim: int, factor: float) -> float:
    return base * (factor ** (dim / (dim - 2)))


def rope_table(dim: int, max_len: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """fp32 ``[max_len, dim/2, 2]`` table of (cos, sin)."""
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    ang = torch.outer(torch.arange(max_len, dtype=torch.float64, device=device), inv).float()
    return torch.stack([torch.cos(ang), torch.sin(ang)], dim=-1).contiguous()


def apply_rope_reference(x: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    """x: [B, S, H, D]; cs: [B, S, D/2, 2] (already indexed by position)."""
    xf = x.float().reshape(*x.shape[:-1], -1, 2)
    c = cs[..., 0].unsqueeze(2)
    s = cs[..., 1].unsqueeze(2)
    x0, x1 = xf[..., 0], xf[..., 1]
    out = torch.stack([x0 * c - x1 * s, x0 * s + x1 * c], dim=-1)
    return out.flatten(-2).to(x.dtype)


def rope_inplace(buf: torch.Tensor, col0: int, n_heads: int, head_dim: int, table: torch.Tensor,
                 positions: Optional[torch.Tensor], seq_len: int, inverse: bool = False,
                 rot_dim: Optional[int] = None, rot_off: int = 0) -> None:
    """Rotate heads stored in ``buf[:, col0 : col0 + n_heads*head_dim]`` in place (CUDA).

    ``positions`` is an int32 tensor with one entry per row of ``buf`` or None
    (then row ``r`` has position ``r % seq_len``). ``rot_dim``/``rot_off``
    restrict the rotation to a slice of each head (MLA rope part).
    """
    rd = head_dim if rot_dim is None else rot_dim
    native().rope_(buf, col0, n_heads, head_dim, positions, seq_len, table, inverse, rd, rot_off)


ROPE_SCALING_METHODS = ("linear", "yarn")


def scaled_rope_table(dim: int, max_len: int, base: float = 10000.0, method: str = "linear", factor: float = 1.0,
                      original_max_len: Optional[int] = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                      attention_factor: Optional[float] = None, device=None) -> torch.Tensor:
    """fp32 ``[max_len, dim/2, 2]`` (cos, sin) table for contexts ``factor`` times longer than trained.

    * ``linear``: position interpolation, every angle divided by ``factor``.
    * ``yarn`` (Peng et al., "YaRN: Efficient Context Window Extension of Large Language Models", 2023):
      pairs up to the one that turns ``beta_fast`` times over ``original_max_len`` positions are left alone,
      those from the one that turns ``beta_slow`` times on are interpolated. Between the two, rounded
      outwards to whole pairs and clamped to [0, dim - 1], the mix is linear in the pair's index, as in the
      tables that published checkpoints run with (the paper's text has it linear in the number of turns).
      (cos, sin) are multiplied by ``attention_factor`` (None: ``0.1 ln(factor) + 1``, and 1 for factors up
      to 1), which scales the scores by its square. The table is then no pure rotation.
    """
    if method not in ROPE_SCALING_METHODS:
        raise ValueError(f"method must be one of {ROPE_SCALING_METHODS}, got {method!r}")
    if factor <= 0:
        raise ValueError(f"factor must be positive, got {factor}")
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    gain = 1.0
    if method == "linear":
        inv = inv / factor
    else:
        if not original_max_len or original_max_len < 0 or not beta_fast > beta_slow > 0 or base <= 1:
            raise ValueError("yarn needs original_max_len, beta_fast > beta_slow > 0 and a base above 1")

        def pair_of(turns):  # where original_max_len * base^(-2i / dim) / (2 pi) = turns
            return dim * math.log(original_max_len / (2 * math.pi * turns)) / (2 * math.log(base))

        low = min(max(math.floor(pair_of(beta_fast)), 0), dim - 1)
        high = min(max(math.ceil(pair_of(beta_slow)), 0), dim - 1)
        pair = torch.arange(dim // 2, dtype=torch.float64, device=device)
        keep = 1 - ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        inv = inv / factor * (1 - keep) + inv * keep
        gain = attention_factor if attention_factor is not None else 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    ang = torch.outer(torch.arange(max_len, dtype=torch.float64, device=device), inv)
    return (gain * torch.stack([torch.cos(ang), torch.sin(ang)], dim=-1)).float().contiguous()
