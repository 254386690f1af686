"""Paged KV cache in 8-bit integers with one magnitude for each block of tokens and head.

The reference's cache holds the model's type (astrai/inference/core/cache.py:189-276); here a token and
head take ``head_dim`` bytes for k and as many for v, half of bfloat16, and decode attention, which is
bound by reading the cache, moves half the bytes.

A :class:`KV8` holds, for pages ``[n_pages, n_kv_heads, page_size, head_dim]``, the integers ``q`` in
[-127, 127] and the largest magnitude ``absmax`` of each ``block`` of tokens of a page and head; a value
is ``q * absmax / 127``.

* :func:`kv8_append`    quantises new tokens ``starts[b] .. lens[b] - 1`` of each row into its pages
* :func:`kv8_attention` causal attention of the row's last tokens over the cache
* :func:`kv8_gather`    the values of a range of tokens, contiguous (for the prefill attention kernel)

Rows are described as everywhere in the framework: an int32 page table ``[B, max_pages]`` (-1: no page)
and int32 lengths on the device, so no call waits for the GPU. On CUDA the kernels of ``csrc/kv8.cu``
run (bfloat16 and float16, head_dim 64 or 128, blocks of 16, 32, 64 or 128 tokens); CPU tensors take
the plain PyTorch functions below.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from astrai_b200.ops._ext import native

BLOCKS = (16, 32, 64, 128)


class KV8(NamedTuple):
    """One layer's 8-bit cache: int8 values and fp32 block magnitudes of k and v."""

    k: torch.Tensor          # int8 [n_pages, n_kv_heads, page_size, head_dim]
    v: torch.Tensor
    k_absmax: torch.Tensor   # fp32 [n_pages, n_kv_heads, page_size / block]
    v_absmax: torch.Tensor

    @classmethod
    def allocate(cls, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, block: int = 32,
                 device=None) -> "KV8":
        if block not in BLOCKS or page_size % block:
            raise ValueError(f"block must be one of {BLOCKS} and divide page_size {page_size}, got {block}")
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        mags = (n_pages, n_kv_heads, page_size // block)
        return cls(*(torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2)),
                   *(torch.zeros(mags, dtype=torch.float32, device=device) for _ in range(2)))

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def block(self) -> int:
        return self.k.shape[2] // self.k_absmax.shape[2]


# ----------------------------------------------------------------------------- append
@torch.no_grad()
def _append_reference(cache: KV8, k, v, page_table, starts, lens) -> None:
    block, page = cache.block, cache.page_size
    S = k.shape[1]
    for b, (first, end) in enumerate(zip(starts.tolist(), lens.tolist())):
        start, end = max(first, 0), min(end, first + S)
        for base in range(start // block * block, end if end > start else 0, block):
            lp = base // page
            p = int(page_table[b, lp]) if lp < page_table.shape[1] else -1
            if not 0 <= p < cache.k.shape[0]:
                continue
            off, kept, stop = base % page, max(0, start - base), min(end - base, block)
            for q, absmax, new in ((cache.k, cache.k_absmax, k), (cache.v, cache.v_absmax, v)):
                x = new[b, base + kept - first: base + stop - first].float().transpose(0, 1)  # [Hkv, n, D]
                fresh = x.abs().amax((1, 2))
                was = absmax[p, :, off // block].clone() if kept else torch.zeros_like(fresh)
                now = torch.where(torch.isfinite(fresh), torch.maximum(was, fresh), math.nan)
                by = torch.where(now > 0, now, 1.0)[:, None, None].double()
                if kept:
                    old = q[p, :, off: off + kept]
                    grown = torch.round(old.double() * was[:, None, None].double() / by).to(torch.int8)
                    old.copy_(torch.where((now > was)[:, None, None], grown, old))
                qx = torch.round(x.double() * 127 / by).clamp(-127, 127)
                q[p, :, off + kept: off + stop] = torch.where((now > 0)[:, None, None], qx, 0).to(torch.int8)
                absmax[p, :, off // block] = now


def kv8_append(cache: KV8, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
               lens: torch.Tensor) -> None:
    """Quantise new tokens into the cache, in place.

    k, v ``[B, S, n_kv_heads, head_dim]`` (any strides with 16-byte aligned rows, e.g. slices of the QKV
    projection). Row ``b`` keeps its tokens before ``starts[b]`` and gets ``lens[b] - starts[b]`` (at most
    S) new ones, ``k[b, i]`` at position ``starts[b] + i``; what the cache held from ``starts[b]`` on is
    void. A block that held earlier tokens ends under the larger of the two magnitudes, and its integers
    are rounded again when that grew. Tokens before position 0 and tokens whose page is missing are
    dropped. A block with an infinity or NaN among its new values reads as NaN. No page may be in the
    table twice. No gradient reaches k and v through the cache.
    """
    if cache.k.is_cuda:
        native().kv8_append(k, v, *cache, page_table, starts, lens)
    else:
        _append_reference(cache, k, v, page_table, starts, lens)


# ----------------------------------------------------------------------------- read-back
def kv8_gather(cache: KV8, page_table: torch.Tensor, lens: torch.Tensor, total: int,
               starts: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Values of tokens ``starts[b] .. starts[b] + total - 1`` (None: from 0) -> k, v
    ``[B, total, n_kv_heads, head_dim]``; zeros from ``lens[b]`` on and where a page is missing."""
    if cache.k.is_cuda:
        return native().kv8_gather(*cache, page_table, starts, lens, total, dtype)
    B = page_table.shape[0]
    page, block = cache.page_size, cache.block
    pos = torch.arange(int(total)) + (0 if starts is None else starts.long()[:, None]) + torch.zeros(B, 1, dtype=torch.long)
    where = pos.clamp(min=0) // page
    pages = page_table.long().gather(1, where.clamp(max=page_table.shape[1] - 1))
    ok = (pos >= 0) & (pos < lens.long()[:, None]) & (where < page_table.shape[1]) & (pages >= 0) \
        & (pages < cache.k.shape[0])
    p, off = torch.where(ok, pages, 0), pos.clamp(min=0) % page
    out = []
    for q, absmax in ((cache.k, cache.k_absmax), (cache.v, cache.v_absmax)):
        x = q[p, :, off].float() * (absmax[p, :, off // block] / 127)[..., None]
        out.append(x.masked_fill(~ok[..., None, None], 0).to(dtype))
    return out[0], out[1]


# ----------------------------------------------------------------------------- attention
def _attention_reference(q, cache: KV8, page_table, lens, starts, scale) -> torch.Tensor:
    B, S, Hq, D = q.shape
    total = page_table.shape[1] * cache.page_size
    k, v = kv8_gather(cache, page_table, lens, total, dtype=torch.float32)
    G = Hq // k.shape[2]
    first = lens.long() - S if starts is None else starts.long()
    pos = first[:, None] + torch.arange(S)
    where = torch.arange(total) // cache.page_size
    held = (page_table >= 0) & (page_table < cache.k.shape[0])
    seen = (torch.arange(total) <= pos[..., None]) & (torch.arange(total) < lens[:, None, None]) \
        & ((pos >= 0) & (pos < lens[:, None]))[..., None] & held[:, where][:, None]
    s = torch.einsum("bshd,bkhd->bhsk", q.float(), k.repeat_interleave(G, 2)) * scale
    p = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
    p = torch.where(seen.any(-1)[:, None, :, None], p, 0.0)
    v = v.repeat_interleave(G, 2)
    bad = ~torch.isfinite(v)
    o = torch.einsum("bhsk,bkhd->bshd", p, v.masked_fill(bad, 0.0))
    if bad.any():  # a weight of 0 would not keep what is not finite out of a sum
        o = o.masked_fill(torch.einsum("bsk,bkhd->bshd", seen.float(), bad.float()) > 0, math.nan)
    return o.to(q.dtype)


def kv8_attention(q: torch.Tensor, cache: KV8, page_table: torch.Tensor, lens: torch.Tensor,
                  starts: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each row's newest tokens over its cached ones -> ``[B, S, n_heads, head_dim]``.

    q ``[B, S, n_heads, head_dim]`` (any strides with 16-byte aligned rows); ``lens[b]`` tokens are cached,
    the queries' own among them. Query ``i`` of row ``b`` has position ``starts[b] + i`` (None:
    ``lens[b] - S + i``) and sees the keys up to its own; a query at or past ``lens[b]``, before token 0, or
    with no page to read gives zeros. Query head ``h`` reads KV head ``h // (n_heads // n_kv_heads)``.
    ``scale`` defaults to ``1 / sqrt(head_dim)``. ``workspace`` fp32 of :func:`kv8_attention_workspace`
    elements is used if given (a caller that captures graphs keeps one per stream); otherwise one is
    allocated. On CUDA it has no gradient: under grad mode a query that requires one is refused, and so is a
    tangent.
    """
    sc = float(scale) if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if not cache.k.is_cuda:
        return _attention_reference(q, cache, page_table, lens, starts, sc)
    return native().kv8_attend(q, *cache, page_table, lens, starts, workspace, sc)


def kv8_attention_workspace(batch: int, tokens: int, n_heads: int, cache: KV8, max_pages: int) -> int:
    """fp32 elements of workspace that :func:`kv8_attention` uses for these sizes."""
    return int(native().kv8_attend_workspace(batch, tokens, n_heads, cache.k.shape[1], cache.k.shape[3],
                                             cache.page_size, max_pages, cache.k.device.index or 0))
