"""The operators as registered PyTorch ops: ``torch.ops.flashprefill.prefill_dense`` and
``torch.ops.flashprefill.prefill_varlen``, and for the paged cache ``kv_cache_write``, ``kv_cache_read`` and
``paged_decode`` of the same namespace.

They wrap the same C ABI entry points as ``flash_prefill`` / ``flash_prefill_varlen_func``
(``fpb_prefill_dense`` / ``fpb_prefill_varlen``), each writing its output argument in place.
They are registered with fake (meta) implementations, so ``torch.compile`` and other graph
tracing can follow a model that calls them without a graph break.  The reference calls its
Python functions directly; these ops take the same positional arguments.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _ops, paged_cache

_NS = "flashprefill"


@torch.library.custom_op(f"{_NS}::prefill_dense", mutates_args=("out",), device_types="cuda")
def prefill_dense(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, block_size: int,
                  attention_sink: int, window_size: int, alpha: float, last_n_block_full: int,
                  min_budget: int) -> None:
    """flash_prefill (ops/flashprefill_native_forward.py:481-499) as a registered op."""
    _ops.prefill_dense(q, k, v, out, block_size, attention_sink, window_size, alpha, last_n_block_full,
                       min_budget)


@prefill_dense.register_fake
def _(q, k, v, out, block_size, attention_sink, window_size, alpha, last_n_block_full, min_budget):
    return None


@torch.library.custom_op(f"{_NS}::prefill_varlen", mutates_args=("o",), device_types="cuda")
def prefill_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, cu_seqlens: torch.Tensor,
                   max_seq_len: int, alpha: float, block_size: int = 128, attention_sink: int = 2,
                   window_size: int = 4, last_n_block: int = 2) -> None:
    """flash_prefill_varlen_func (ops/flashprefill_varlen_func.py:723-743) as a registered op."""
    _ops.prefill_varlen(q, k, v, o, cu_seqlens, max_seq_len, alpha, block_size, attention_sink, window_size,
                        last_n_block)


@prefill_varlen.register_fake
def _(q, k, v, o, cu_seqlens, max_seq_len, alpha, block_size=128, attention_sink=2, window_size=4,
      last_n_block=2):
    return None


@torch.library.custom_op(f"{_NS}::kv_cache_write", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"),
                         device_types="cuda")
def kv_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                   k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor]) -> None:
    """paged_cache.kv_cache_write as a registered op (what it writes is given: None scales for a 16-bit cache)."""
    paged_cache.kv_cache_write(k, v, k_cache, v_cache, slots, k_scale, v_scale)


@kv_cache_write.register_fake
def _(k, v, k_cache, v_cache, slots, k_scale, v_scale):
    return None


@torch.library.custom_op(f"{_NS}::kv_cache_read", mutates_args=("k", "v"), device_types="cuda")
def kv_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                  k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                  v_scale: Optional[torch.Tensor] = None) -> None:
    """paged_cache.kv_cache_read as a registered op."""
    paged_cache.kv_cache_read(k_cache, v_cache, page_table, seq_lens, k, v, k_scale, v_scale)


@kv_cache_read.register_fake
def _(k_cache, v_cache, page_table, seq_lens, k, v, k_scale=None, v_scale=None):
    return None


@torch.library.custom_op(f"{_NS}::paged_decode", mutates_args=("out", "lse"), device_types="cuda")
def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, out: torch.Tensor, lse: Optional[torch.Tensor],
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                 sm_scale: Optional[float] = None) -> None:
    """paged_cache.paged_decode as a registered op (its workspace from the caching allocator)."""
    paged_cache.paged_decode(q, k_cache, v_cache, page_table, seq_lens, out, lse, k_scale, v_scale, sm_scale)


@paged_decode.register_fake
def _(q, k_cache, v_cache, page_table, seq_lens, out, lse, k_scale=None, v_scale=None, sm_scale=None):
    return None
