"""Serving: a paged key/value cache of ragged sequences, and attention over it.

    cuda_attn.paged_append(k, v, k_cache, v_cache, page_table, kv_lens, cu_new)
    o = cuda_attn.paged_attn(q, k_cache, v_cache, page_table, kv_lens, cu_new, max_new=n)

The caches are pools of pages, (pages, heads, page size, d), of which each sequence has the ones in its row of `page_table`
(batch, width): its token t is in page page_table[b, t // page size] at place t % page size. `kv_lens[b]` tokens of it are
cached. A call's new tokens, the last ones of each sequence, are packed one sequence after another in (tokens, heads, d)
tensors: those of sequence b are rows cu_new[b] to cu_new[b + 1], and kv_lens counts them. The three are int32 tensors on
the GPU; no call waits for the GPU, so a decoding step can be captured in a CUDA graph and replayed as they change.

Caches are float16 or bfloat16, the type of the new tokens, or int8 with `k_scale` and `v_scale`, float32 (pages, heads,
page size): a vector x of one token and head is held as round(127 x / top) and top / 127, top = max |x| (at least
127 * 2^-100). Head dimension 64 or 128, page sizes 16, 32, ... 1024, 1 to 128 query heads for each key head. Strided views
are taken as they are (a slice of a fused projection, a pool that holds keys and values interleaved) where their strides
are multiples of 16 bytes and d is contiguous.

A page id, length or offset that is out of range is not followed: the token is not written, reads as zeros (to the
attention, under a page id out of range, as a key and a value of zeros; past its row's room as no key at all), and
device_status() says so (bit 512). Packed tokens after cu_new[-1] are of no sequence and get zeros, and so do those before
cu_new[0], which should be 0.
"""
from __future__ import annotations

import ctypes

import torch

from . import _ext  # defined above this module's import in the package


def paged_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                 kv_lens: torch.Tensor, cu_new: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None) -> None:
    """Write the new tokens' keys and values (tokens, heads, d) into the cache, quantised if it is int8."""
    _ext().paged_append(k, v, k_cache, v_cache, page_table, kv_lens, cu_new, k_scale, v_scale)


def paged_read(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
               cu_new: torch.Tensor, total: int, dtype: torch.dtype | None = None, k_scale: torch.Tensor | None = None,
               v_scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values (total, heads, d) that the cache holds of the last cu_new[b + 1] - cu_new[b] tokens of each
    sequence; all of them where that is kv_lens[b]. `total` is cu_new[-1], known to the caller. `dtype`: the cache's, or
    float16 or bfloat16 of an int8 cache (bfloat16 by default)."""
    if dtype is None:
        dtype = torch.bfloat16 if k_cache.dtype == torch.int8 else k_cache.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"paged_read: dtype must be float16 or bfloat16 (got {dtype})")
    return _ext().paged_read(k_cache, v_cache, page_table, kv_lens, cu_new, total, dtype == torch.bfloat16, k_scale, v_scale)


def paged_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
               kv_lens: torch.Tensor, cu_new: torch.Tensor, k_scale: torch.Tensor | None = None,
               v_scale: torch.Tensor | None = None, causal: bool = True, max_new: int = 0,
               scale: float | None = None) -> torch.Tensor:
    """Attention of the new tokens' queries (tokens, query heads, d) over all cached tokens of their sequences (append
    their keys and values first). Query head h reads key head h // (query heads / heads); new token i of n sees the first
    kv_lens[b] - n + i + 1 tokens if causal, else all kv_lens[b]; one that sees none gets zeros. `scale` of the scores: 1 /
    sqrt(d) by default. `max_new`: the largest number of new tokens of a sequence, a hint that picks the kernel, and with it
    the speed and the rounding (default: the average). The same call repeats bit for bit; the last bits also depend on the
    other sequences of the batch and on page_table's width. 16-bit values within kv_lens[b] must be finite, those that the
    causal mask hides too; a NaN among the keys, or in an int8 cache, reaches the rows that see it alone. What the pages
    hold past kv_lens[b] may be anything."""
    if scale is not None and not 0.0 < abs(ctypes.c_float(scale).value) < float("inf"):
        raise RuntimeError(f"paged_attn: scale must be finite and not zero in float32 (got {scale})")
    return _ext().paged_attn(q, k_cache, v_cache, page_table, kv_lens, cu_new, k_scale, v_scale, causal, max_new,
                             0.0 if scale is None else scale)
