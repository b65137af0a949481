"""Paged key/value cache and decode attention: what follows a prefill.

``flash_prefill`` answers for a whole prompt; these entry points keep its keys and values in pages and attend to them one
token at a time.  The reference has no counterpart (its callers hand decode to their host framework,
patches/patch_loader_vllm_0_12_0.py:167-168).

A cache is a pair of tensors (num_pages, page_size, kv_heads, 128) that share strides (any, with rows of 128 contiguous
elements at multiples of 16 bytes): token-major pages as vLLM keeps them, or head-major as ``kv_cache_alloc`` makes them.  It holds the
rows' 16-bit type, or ``torch.float8_e4m3fn`` codes with a float32 scale for each (token, head) in ``k_scale`` and ``v_scale``
(num_pages, page_size, kv_heads).  A sequence's token s lives at ``page_table[b, s // page_size]``, offset ``s % page_size``;
its slot is ``page * page_size + offset``.

All calls are asynchronous on the current stream, allocate nothing but a decode call's workspace, never synchronise, and
can be captured in a CUDA graph.  Slots, pages and lengths are checked on the device: one that points outside its tensors is skipped and
reported by ``check_paged_error``, which waits for the current stream and clears what all calls on the device have met (with
FLASHPREFILL_B200_CHECK=1 by the call itself, which then runs alone; a captured call reports to whoever checks after its replay).
Shapes, types and strides that are not supported raise ValueError or TypeError.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, _ops


class KVCache(NamedTuple):
    """The tensors of a paged cache; the scales are None for a 16-bit cache."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None
    v_scale: torch.Tensor | None


def kv_cache_alloc(num_pages: int, page_size: int, kv_heads: int, dtype: torch.dtype = torch.bfloat16,
                   device="cuda") -> KVCache:
    """A cache with head-major pages (a page's rows of one head are contiguous, which decode reads fastest), uninitialised:
    the values of rows that were never written do not reach any result.  ``dtype``: bfloat16, float16 or float8_e4m3fn."""
    if dtype not in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
        raise TypeError(f"a cache holds bfloat16, float16 or float8_e4m3fn (got {dtype})")
    if num_pages < 1 or page_size < 1 or kv_heads < 1:
        raise ValueError("num_pages, page_size and kv_heads must be >= 1")
    rows = lambda: torch.empty(num_pages, kv_heads, page_size, 128, dtype=dtype, device=device).transpose(1, 2)
    scales = lambda: torch.empty(num_pages, kv_heads, page_size, dtype=torch.float32, device=device).transpose(1, 2)
    if dtype is torch.float8_e4m3fn:
        return KVCache(rows(), rows(), scales(), scales())
    return KVCache(rows(), rows(), None, None)


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                   k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """Write rows k, v (T, kv_heads, 128) into the cache slots ``slots`` (T,), int64 or int32; a negative slot skips its row.

    An e4m3 cache gets ``scale = max(max|x|, 2**-100) / 448`` and codes ``x * (448 / max(max|x|, 2**-100))`` for each row; a row with an infinity or
    a NaN reads back as NaN.  k and v may have any strides (e.g. columns of a fused projection; copied only where rows are not
    16-byte aligned).  The slots of one call must differ from one another (FLASHPREFILL_B200_CHECK=1 checks that); where two
    rows name one slot, its contents are not defined.  k_cache and v_cache must be different memory, as must the scales."""
    write = (_lib._ext or _lib.ext()).kv_cache_write
    if _ops.CHECK:
        return _ops.checked_paged(write, (k, v, k_cache, v_cache, slots, k_scale, v_scale), slots)
    write(k, v, k_cache, v_cache, slots, k_scale, v_scale)


def kv_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                  k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                  v_scale: torch.Tensor | None = None) -> None:
    """Copy the first ``seq_lens[b]`` cached rows of every sequence into k, v (B, S, kv_heads, 128), the layout that
    ``flash_prefill`` takes for a cached prefix, dequantising an e4m3 cache to their 16-bit type.  Rows from ``seq_lens[b]`` on
    are left as they were, as is all of a sequence whose length is outside [0, S].  page_table (B, P) and seq_lens (B,) are
    int32."""
    read = (_lib._ext or _lib.ext()).kv_cache_read
    if _ops.CHECK:
        return _ops.checked_paged(read, (k_cache, v_cache, page_table, seq_lens, k, v, k_scale, v_scale))
    read(k_cache, v_cache, page_table, seq_lens, k, v, k_scale, v_scale)


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, out: torch.Tensor, lse: torch.Tensor | None = None,
                 k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, sm_scale: float | None = None,
                 workspace: torch.Tensor | None = None) -> None:
    """Attention of one new token for each sequence, q (B, q_heads, 128), over its ``seq_lens[b]`` cached tokens (write the new
    token's own row first); GQA with q_heads a multiple of kv_heads.  Writes ``out`` (like q) in place and, if given, ``lse``
    (B, q_heads) float32: log sum exp(sm_scale q.k), with which outputs over parts of a sequence can be joined.

    A sequence of length 0 gives zeros and -inf, as does one whose length is outside [0, P * page_size].  Infinite values of a
    16-bit cache keep to the softmax (any weight makes the channel infinite; a weight that vanishes, below 2^-39 of the largest
    for float16 and 2^-100 for bfloat16, makes it NaN, as 0 times infinity).  Weights meet the values with 16 bits or more; with 11,
    an eighth of the output's rounding, where an e4m3 cache is answered in bfloat16.  ``sm_scale`` is 1/sqrt(128) by default.  ``workspace``: uint8 of at least ``paged_decode_workspace_bytes``, taken from the caching
    allocator by default; calls that may overlap on the GPU (other streams, graphs replayed side by side) need one each.
    Results do not depend on the order in which the GPU runs its blocks: the same call gives the same bits (the same sequences
    behind a table of another width may be split, and rounded, in another way)."""
    decode = (_lib._ext or _lib.ext()).paged_decode
    if _ops.CHECK:
        return _ops.checked_paged(decode, (q, k_cache, v_cache, page_table, seq_lens, out, lse, k_scale, v_scale, sm_scale, workspace))
    decode(q, k_cache, v_cache, page_table, seq_lens, out, lse, k_scale, v_scale, sm_scale, workspace)
