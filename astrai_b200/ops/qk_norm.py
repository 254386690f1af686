"""RMS norm of every query and key head together with the rotation of its position.

The reference rotates q and k with elementwise ops and then normalises each head
(astrai/model/components/rope.py:26-33, attention.py:79-84). :func:`qk_norm_rope` does both in one
pass over the fused projection output, forward and backward, and knows what other checkpoints need:
the norm before the rotation, the half layout (channel ``i`` rotates with ``i + rot_dim / 2``),
a rotation of part of each head, and tables scaled for long contexts
(:func:`astrai_b200.ops.rope.scaled_rope_table`).

With ``z`` one head, ``R`` the rotation and ``n(z) = z / sqrt(mean z^2 + eps) * w``:

* ``norm="after"``  ``y = n(R x)`` (the reference's order)
* ``norm="before"`` ``y = R n(x)``
* ``norm="none"``   ``y = R x``

On CUDA bfloat16, float16 and float32 run on the kernels of ``csrc/qk_norm.cu`` (fp32 inside, one
rounding at the end); CPU tensors take the plain PyTorch math of :func:`qk_norm_rope_reference`.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from astrai_b200.ops._ext import native

NORM_MODES = {"none": 0, "after": 1, "before": 2}
LAYOUTS = ("interleaved", "half")


def rotate_reference(x: torch.Tensor, cs: torch.Tensor, layout: str, rot_dim: int, rot_off: int = 0) -> torch.Tensor:
    """x ``[..., H, D]`` rotated in its own type; cs ``[..., rot_dim / 2, 2]``, one row per token."""
    c, s = cs[..., 0].unsqueeze(-2), cs[..., 1].unsqueeze(-2)
    part = x[..., rot_off: rot_off + rot_dim]
    if layout == "half":
        a, b = part.chunk(2, -1)
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([x[..., :rot_off], turned, x[..., rot_off + rot_dim:]], -1)


def qk_norm_rope_reference(x, n_heads, n_kv_heads, head_dim, table, q_weight=None, k_weight=None, positions=None,
                           seq_len=None, eps=1e-6, layout="interleaved", norm="after", rot_dim=None, rot_off=0):
    """Plain PyTorch math (at least fp32, rounded once); same arguments as :func:`qk_norm_rope`."""
    rot = head_dim if rot_dim is None else rot_dim
    H = n_heads + n_kv_heads
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    z = x[:, : H * head_dim].to(wide).reshape(-1, H, head_dim)
    if positions is None:
        positions = torch.arange(z.shape[0], device=x.device) % seq_len
    cs = table.to(wide)[positions.reshape(-1).long()]
    if norm != "none":
        w = torch.cat([q_weight.to(wide).expand(n_heads, head_dim), k_weight.to(wide).expand(n_kv_heads, head_dim)])

    def n(t):
        return t * torch.rsqrt((t * t).mean(-1, keepdim=True) + eps) * w

    if norm == "before":
        z = n(z)
    z = rotate_reference(z, cs, layout, rot, rot_off)
    if norm == "after":
        z = n(z)
    return z.reshape(-1, H * head_dim).to(x.dtype)


def _check(x, n_heads, n_kv_heads, head_dim, table, q_weight, k_weight, positions, seq_len, layout, norm, rot, off):
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if norm not in NORM_MODES:
        raise ValueError(f"norm must be one of {tuple(NORM_MODES)}, got {norm!r}")
    if x.dim() != 2 or x.shape[1] < (n_heads + n_kv_heads) * head_dim:
        raise ValueError(f"x must be [rows, >= {(n_heads + n_kv_heads) * head_dim}], got {tuple(x.shape)}")
    if rot <= 0 or rot % 2 or off < 0 or rot + off > head_dim:
        raise ValueError(f"rot_dim {rot} at offset {off} does not fit an even part of head_dim {head_dim}")
    if table.dim() != 3 or table.shape[1] * 2 != rot or table.shape[2] != 2:
        raise ValueError(f"table must be [max_pos, {rot // 2}, 2], got {tuple(table.shape)}")
    if norm != "none" and (q_weight is None or k_weight is None or q_weight.numel() != head_dim
                           or k_weight.numel() != head_dim):
        raise ValueError(f"norm={norm!r} needs q_weight and k_weight of {head_dim} entries")
    if positions is None and not seq_len:
        raise ValueError("positions or seq_len must be given")
    if positions is not None and positions.numel() != x.shape[0]:
        raise ValueError(f"positions must have one entry per row ({x.shape[0]}), got {positions.numel()}")


def _native(x, n_heads, n_kv_heads, head_dim, table, q_weight, k_weight, positions, seq_len, eps, layout, norm, rot, off,
            in_place):
    """The kernels' call; it checks its arguments itself (csrc/bind_qk_norm.cpp)."""
    mode = NORM_MODES.get(norm)
    if mode is None:
        raise ValueError(f"norm must be one of {tuple(NORM_MODES)}, got {norm!r}")
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    return native().qk_norm_rope(x, n_heads, n_kv_heads, head_dim, table, q_weight, k_weight, positions, seq_len or 0,
                                 eps, layout == "half", mode, rot, off, in_place)


def qk_norm_rope(x: torch.Tensor, n_heads: int, n_kv_heads: int, head_dim: int, table: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, seq_len: Optional[int] = None, eps: float = 1e-6,
                 layout: str = "interleaved", norm: str = "after", rot_dim: Optional[int] = None,
                 rot_off: int = 0) -> torch.Tensor:
    """Normalise and rotate the query and key heads of ``x`` -> ``[rows, (n_heads + n_kv_heads) * head_dim]``.

    ``x`` ``[rows, W]`` holds the query heads, then the key heads, in its first columns (the fused QKV
    projection's output; any row stride; columns behind them are not read). ``table`` is the fp32 (cos,
    sin) table ``[max_pos, rot_dim / 2, 2]``, ``positions`` one integer per row (None: row ``r`` has
    position ``r % seq_len``); a position outside the table leaves its row unrotated and sets the device
    error word. ``rot_dim`` channels from ``rot_off`` are rotated (None: all). On CUDA ``head_dim`` is at
    most 256, and it, ``rot_dim`` and ``rot_off`` are multiples of 8. Differentiable in ``x`` and the
    weights, in reverse mode and once; on CUDA tangents and a table that requires a gradient are refused.
    """
    rot = head_dim if rot_dim is None else rot_dim
    if x.is_cuda:
        return _native(x, n_heads, n_kv_heads, head_dim, table, q_weight, k_weight, positions, seq_len, eps, layout, norm,
                       rot, rot_off, False)
    _check(x, n_heads, n_kv_heads, head_dim, table, q_weight, k_weight, positions, seq_len, layout, norm, rot, rot_off)
    return qk_norm_rope_reference(x, n_heads, n_kv_heads, head_dim, table, q_weight, k_weight, positions, seq_len, eps,
                                  layout, norm, rot, rot_off)


def qk_norm_rope_(x: torch.Tensor, n_heads: int, n_kv_heads: int, head_dim: int, table: torch.Tensor,
                  q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None, seq_len: Optional[int] = None, eps: float = 1e-6,
                  layout: str = "interleaved", norm: str = "after", rot_dim: Optional[int] = None,
                  rot_off: int = 0) -> torch.Tensor:
    """:func:`qk_norm_rope` in place on the query and key columns of ``x`` -> ``x``. It has no gradient: under grad
    mode no input may require one."""
    rot = head_dim if rot_dim is None else rot_dim
    if x.is_cuda:
        return _native(x, n_heads, n_kv_heads, head_dim, table, q_weight, k_weight, positions, seq_len, eps, layout, norm,
                       rot, rot_off, True)
    _check(x, n_heads, n_kv_heads, head_dim, table, q_weight, k_weight, positions, seq_len, layout, norm, rot, rot_off)
    inputs = (x, table) if norm == "none" else (x, table, q_weight, k_weight)
    if torch.is_grad_enabled() and any(t.requires_grad for t in inputs):
        raise RuntimeError("qk_norm_rope_ has no gradient (of x, the weights or the table): use qk_norm_rope")
    x[:, : (n_heads + n_kv_heads) * head_dim] = qk_norm_rope_reference(
        x, n_heads, n_kv_heads, head_dim, table, q_weight, k_weight, positions, seq_len, eps, layout, norm, rot, rot_off)
    return x


@dataclass
class QKRotary:
    """What a layer does to its query and key heads: the arguments of :func:`qk_norm_rope` that do not
    depend on the batch."""

    table: torch.Tensor
    q_weight: Optional[torch.Tensor] = None
    k_weight: Optional[torch.Tensor] = None
    eps: float = 1e-6
    layout: str = "interleaved"
    norm: str = "after"

    @property
    def rot_dim(self) -> int:
        return 2 * self.table.shape[1]

    def _args(self, positions, seq_len) -> dict:
        return dict(table=self.table, q_weight=self.q_weight, k_weight=self.k_weight, positions=positions,
                    seq_len=seq_len, eps=self.eps, layout=self.layout, norm=self.norm, rot_dim=self.rot_dim)

    def apply(self, x, n_heads, n_kv_heads, head_dim, positions=None, seq_len=None) -> torch.Tensor:
        return qk_norm_rope(x, n_heads, n_kv_heads, head_dim, **self._args(positions, seq_len))

    def apply_(self, x, n_heads, n_kv_heads, head_dim, positions=None, seq_len=None) -> torch.Tensor:
        return qk_norm_rope_(x, n_heads, n_kv_heads, head_dim, **self._args(positions, seq_len))

    def kernel_args(self):
        """(weights, rot_dim, rot_off, half layout, norm mode, eps) as the row-buffer kernels take them."""
        w = (None, None) if self.norm == "none" else (self.q_weight, self.k_weight)
        return (*w, self.rot_dim, 0, self.layout == "half", NORM_MODES[self.norm], float(self.eps))
