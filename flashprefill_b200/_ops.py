"""Tensor plumbing between PyTorch and the C ABI: validation, layout, workspace, stream.

PyTorch only provides device memory (the workspace comes from its caching allocator, as
the reference's temporaries do) and the current CUDA stream; all computation happens in
the CUDA kernels of libflashprefill_b200.so.
"""
from __future__ import annotations

import ctypes
import os

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.FPB_BF16, torch.float16: _lib.FPB_FP16}

# Reduction order of the pooled-key sum: the Triton warp count whose order is reproduced
# (the reference's autotuner picks 4 or 8, ops/flashprefill_native_forward.py:7-20).
_MEAN_WARPS = int(os.environ.get("FLASHPREFILL_B200_MEAN_WARPS", "4"))
# When set, every call synchronises and raises if a kernel reported a device error.
_CHECK = os.environ.get("FLASHPREFILL_B200_CHECK", "0") not in ("", "0")

LAYOUT_KEYS = ["err", "cu_tile", "mk", "cnt", "idx", "total", "tiles", "cap"]


def set_mean_warps(w: int) -> None:
    """Choose the pooled-key summation order (4 or 8 warps of Triton's reduction)."""
    global _MEAN_WARPS
    if w not in (4, 8):
        raise ValueError("mean warps must be 4 or 8")
    _MEAN_WARPS = w


def get_mean_warps() -> int:
    return _MEAN_WARPS


def _dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"flashprefill_b200 supports bfloat16 and float16 inputs (got {t.dtype})") from None


def _tma_ok(t: torch.Tensor) -> bool:
    """Can the kernels address t directly (last dim contiguous, 16-byte strides/base)?"""
    if t.stride(-1) != 1 or t.data_ptr() % 16 != 0:
        return False
    return all(s % 8 == 0 for s in t.stride()[:-1])


def _prep_input(t: torch.Tensor, name: str, ndim: int, device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got shape {tuple(t.shape)}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (flashprefill_b200 has no CPU path), got {t.device}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t if _tma_ok(t) else t.contiguous()


def _strides(t: torch.Tensor, n: int):
    return _lib.i64arr(t.stride()[:n])


def _P(x):
    return ctypes.c_void_p(x.data_ptr() if isinstance(x, torch.Tensor) else x)


def _finish(ws: torch.Tensor, stream) -> None:
    if _CHECK:
        check_device_error(ws, stream)


def check_device_error(ws: torch.Tensor, stream=None) -> int:
    """Synchronise and raise if the kernels recorded an error in the workspace."""
    lib = _lib.load()
    if stream is None:
        stream = torch.cuda.current_stream(ws.device).cuda_stream
    flags = ctypes.c_uint32(0)
    rc = lib.fpb_read_device_error(ctypes.c_void_p(ws.data_ptr()), ctypes.byref(flags), ctypes.c_void_p(stream))
    if rc == _lib.FPB_EDEVICE:
        what = [m for b, m in _lib.DEV_ERROR_BITS.items() if flags.value & b]
        raise _lib.FlashPrefillError("flashprefill_b200 device error: " + "; ".join(what))
    _lib.check(rc)
    return flags.value


def dense_layout(batch, seqlen, hq, hk):
    out = (ctypes.c_int64 * 8)()
    _lib.check(_lib.load().fpb_workspace_layout(0, batch, seqlen, 0, hq, hk, 128, out))
    return dict(zip(LAYOUT_KEYS, list(out)))


def varlen_layout(nseq, total, max_seq_len, hq, hk):
    out = (ctypes.c_int64 * 8)()
    _lib.check(_lib.load().fpb_workspace_layout(1, nseq, total, max_seq_len, hq, hk, 128, out))
    return dict(zip(LAYOUT_KEYS, list(out)))


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def _views(ws, L, Hq, Hk, dtype):
    tiles, cap = int(L["tiles"]), int(L["cap"])
    cnt = ws[L["cnt"]:L["cnt"] + 4 * Hq * tiles].view(torch.int32).view(Hq, tiles)
    idx = ws[L["idx"]:L["idx"] + 4 * Hq * tiles * cap].view(torch.int32).view(Hq, tiles, cap)
    mk = ws[L["mk"]:L["mk"] + 2 * tiles * Hk * 128].view(dtype).view(tiles, Hk, 128)
    return cnt, idx, mk


# --------------------------------------------------------------------------- dense
def _dense_args(q, k, v, out, allow_chunk=False):
    device = q.device
    q = _prep_input(q, "q", 4, device)
    k = _prep_input(k, "k", 4, device)
    v = _prep_input(v, "v", 4, device) if v is not None else None
    B, S, Hq, D = q.shape
    if k.shape[0] != B or k.shape[3] != D or not (k.shape[1] == S or (allow_chunk and k.shape[1] > S)):
        raise ValueError(f"k shape {tuple(k.shape)} does not match q shape {tuple(q.shape)}")
    if v is not None and v.shape != k.shape:
        raise ValueError(f"v shape {tuple(v.shape)} must equal k shape {tuple(k.shape)}")
    if k.dtype != q.dtype or (v is not None and v.dtype != q.dtype):
        raise TypeError("q, k and v must share one dtype")
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype or out.device != device:
            raise ValueError("out must be a tensor with q's shape, dtype and device")
    return q, k, v, B, S, Hq, k.shape[2], D


def prefill_dense(q, k, v, out, block_size, attention_sink, window_size, alpha, last_n_block_full, min_budget,
                  workspace: torch.Tensor | None = None, out_peers=None, q_blocks=None):
    """Full operator on (B,S,H,D) tensors; writes ``out`` in place.  Returns the workspace.

    ``out_peers``: device addresses (ints) of the same output slice in other GPUs' copies of
    the output; every output tile is written there too (fpb_prefill_dense_peers).
    ``q_blocks``: (begin, end) query-block range; only those rows are searched and written,
    with the selection rules of the whole sequence (fpb_prefill_dense_rows).
    k/v longer than q: chunked prefill, the queries being the last q.shape[1] positions
    (fpb_prefill_dense_chunk)."""
    lib = _lib.load()
    Skv = k.shape[1] if isinstance(k, torch.Tensor) and k.dim() == 4 else None
    q, k, v, B, S, Hq, Hk, D = _dense_args(q, k, v, out, allow_chunk=True)
    if Skv is not None and Skv != S:
        if out_peers or q_blocks is not None:
            raise ValueError("chunked prefill cannot be combined with out_peers or q_blocks")
        return _prefill_chunk(lib, q, k, v, out, B, S, Skv, Hq, Hk, D, block_size, attention_sink, window_size,
                              alpha, last_n_block_full, min_budget, workspace)
    code = _dtype_code(q)
    tgt = out if _tma_ok(out) else torch.empty_like(q)
    if out_peers and tgt is not out:
        raise ValueError("out must be a TMA-compatible strided view when out_peers is given")
    ws = workspace if workspace is not None else _workspace(lib.fpb_dense_workspace_bytes(B, S, Hq, Hk, D), q.device)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    with torch.cuda.device(q.device):
        args = (_P(q), _P(k), _P(v), _P(tgt), code, B, S, Hq, Hk, D, _strides(q, 3), _strides(k, 3), _strides(v, 3),
                _strides(tgt, 3), int(block_size), int(attention_sink), int(window_size), float(alpha),
                int(last_n_block_full), int(min_budget), _MEAN_WARPS, _P(ws), ws.numel())
        if out_peers and q_blocks is not None:
            raise ValueError("out_peers and q_blocks cannot be combined")
        if out_peers:
            peers = (ctypes.c_void_p * len(out_peers))(*[int(p) for p in out_peers])
            rc = lib.fpb_prefill_dense_peers(*args, peers, len(out_peers), _P(stream))
        elif q_blocks is not None:
            rc = lib.fpb_prefill_dense_rows(*args[:21], int(q_blocks[0]), int(q_blocks[1]), *args[21:], _P(stream))
        else:
            rc = lib.fpb_prefill_dense(*args, _P(stream))
    _lib.check(rc)
    if tgt is not out:
        out.copy_(tgt)
    _finish(ws, stream)
    return ws


def _prefill_chunk(lib, q, k, v, out, B, Sq, Skv, Hq, Hk, D, block_size, attention_sink, window_size, alpha,
                   last_n_block_full, min_budget, workspace):
    code = _dtype_code(q)
    tgt = out if _tma_ok(out) else torch.empty_like(q)
    ws = workspace if workspace is not None else _workspace(lib.fpb_dense_workspace_bytes(B, Skv, Hq, Hk, D), q.device)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    with torch.cuda.device(q.device):
        rc = lib.fpb_prefill_dense_chunk(_P(q), _P(k), _P(v), _P(tgt), code, B, Sq, Skv, Hq, Hk, D, _strides(q, 3),
                                         _strides(k, 3), _strides(v, 3), _strides(tgt, 3), int(block_size),
                                         int(attention_sink), int(window_size), float(alpha), int(last_n_block_full),
                                         int(min_budget), _MEAN_WARPS, _P(ws), ws.numel(), _P(stream))
    _lib.check(rc)
    if tgt is not out:
        out.copy_(tgt)
    _finish(ws, stream)
    return ws


def search_dense(q, k, block_size=128, attention_sink=2, window_size=4, alpha=0.18, last_n_block_full=2,
                 min_budget=0, workspace: torch.Tensor | None = None):
    """Block search only.  Returns (counts [Hq, B*NB] int32, lists [Hq, B*NB, NB] int32,
    pooled keys [B*NB, Hk, D], workspace); row b*NB + qb of head h lists counts[h, row]
    ascending key-block indices."""
    lib = _lib.load()
    q, k, _, B, S, Hq, Hk, D = _dense_args(q, k, None, None)
    code = _dtype_code(q)
    L = dense_layout(B, S, Hq, Hk)
    ws = workspace if workspace is not None else _workspace(L["total"], q.device)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    with torch.cuda.device(q.device):
        rc = lib.fpb_search_dense(_P(q), _P(k), code, B, S, Hq, Hk, D, _strides(q, 3), _strides(k, 3),
                                  int(block_size), int(attention_sink), int(window_size), float(alpha),
                                  int(last_n_block_full), int(min_budget), _MEAN_WARPS, _P(ws), ws.numel(),
                                  _P(stream))
    _lib.check(rc)
    _finish(ws, stream)
    return _views(ws, L, Hq, Hk, q.dtype) + (ws,)


def attention_dense(q, k, v, out, workspace: torch.Tensor, block_size=128):
    """Attention stage only over the block lists held in ``workspace``."""
    lib = _lib.load()
    q, k, v, B, S, Hq, Hk, D = _dense_args(q, k, v, out)
    code = _dtype_code(q)
    tgt = out if _tma_ok(out) else torch.empty_like(q)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    with torch.cuda.device(q.device):
        rc = lib.fpb_attention_dense(_P(q), _P(k), _P(v), _P(tgt), code, B, S, Hq, Hk, D, _strides(q, 3),
                                     _strides(k, 3), _strides(v, 3), _strides(tgt, 3), int(block_size),
                                     _P(workspace), workspace.numel(), _P(stream))
    _lib.check(rc)
    if tgt is not out:
        out.copy_(tgt)
    _finish(workspace, stream)


# --------------------------------------------------------------------------- varlen
def _varlen_args(q, k, v, o, cu_seqlens):
    device = q.device
    q = _prep_input(q, "q", 3, device)
    k = _prep_input(k, "k", 3, device)
    v = _prep_input(v, "v", 3, device) if v is not None else None
    T, Hq, D = q.shape
    if k.shape[0] != T or k.shape[2] != D:
        raise ValueError(f"k shape {tuple(k.shape)} does not match q shape {tuple(q.shape)}")
    if v is not None and v.shape != k.shape:
        raise ValueError("v shape must equal k shape")
    if k.dtype != q.dtype or (v is not None and v.dtype != q.dtype):
        raise TypeError("q, k and v must share one dtype")
    if o is not None and (o.shape != q.shape or o.dtype != q.dtype or o.device != device):
        raise ValueError("o must be a tensor with q's shape, dtype and device")
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise ValueError("cu_seqlens must be a 1-D tensor with at least 2 entries")
    if cu_seqlens.device != device:
        raise ValueError(f"cu_seqlens must be on {device}")
    cu = cu_seqlens if cu_seqlens.dtype == torch.int32 and cu_seqlens.is_contiguous() else \
        cu_seqlens.to(torch.int32).contiguous()
    return q, k, v, cu, T, Hq, k.shape[1], D


def prefill_varlen(q, k, v, o, cu_seqlens, max_seq_len, alpha, block_size=128, attention_sink=2, window_size=4,
                   last_n_block=2, workspace: torch.Tensor | None = None):
    """Full operator on packed (T,H,D) tensors; writes ``o`` in place.  Returns the workspace."""
    lib = _lib.load()
    q, k, v, cu, T, Hq, Hk, D = _varlen_args(q, k, v, o, cu_seqlens)
    code = _dtype_code(q)
    nseq = cu.numel() - 1
    tgt = o if _tma_ok(o) else torch.empty_like(q)
    nbytes = lib.fpb_varlen_workspace_bytes(T, nseq, int(max_seq_len), Hq, Hk, D)
    ws = workspace if workspace is not None else _workspace(nbytes, q.device)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    with torch.cuda.device(q.device):
        rc = lib.fpb_prefill_varlen(_P(q), _P(k), _P(v), _P(tgt), code, _P(cu), nseq, T, int(max_seq_len), Hq, Hk,
                                    D, _strides(q, 2), _strides(k, 2), _strides(v, 2), _strides(tgt, 2),
                                    int(block_size), int(attention_sink), int(window_size), float(alpha),
                                    int(last_n_block), _MEAN_WARPS, _P(ws), ws.numel(), _P(stream))
    _lib.check(rc)
    if tgt is not o:
        o.copy_(tgt)
    _finish(ws, stream)
    return ws


def search_varlen(q, k, cu_seqlens, max_seq_len, alpha, block_size=128, attention_sink=2, window_size=4,
                  last_n_block=2, workspace: torch.Tensor | None = None):
    """Block search only.  Returns (counts [Hq, tiles], lists [Hq, tiles, cap], pooled keys,
    cu_tile [nseq+1], workspace)."""
    lib = _lib.load()
    q, k, _, cu, T, Hq, Hk, D = _varlen_args(q, k, None, None, cu_seqlens)
    code = _dtype_code(q)
    nseq = cu.numel() - 1
    L = varlen_layout(nseq, T, int(max_seq_len), Hq, Hk)
    ws = workspace if workspace is not None else _workspace(L["total"], q.device)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    with torch.cuda.device(q.device):
        rc = lib.fpb_search_varlen(_P(q), _P(k), code, _P(cu), nseq, T, int(max_seq_len), Hq, Hk, D,
                                   _strides(q, 2), _strides(k, 2), int(block_size), int(attention_sink),
                                   int(window_size), float(alpha), int(last_n_block), _MEAN_WARPS, _P(ws),
                                   ws.numel(), _P(stream))
    _lib.check(rc)
    _finish(ws, stream)
    cnt, idx, mk = _views(ws, L, Hq, Hk, q.dtype)
    cu_tile = ws[L["cu_tile"]:L["cu_tile"] + 4 * (nseq + 1)].view(torch.int32)
    return cnt, idx, mk, cu_tile, ws


def attention_varlen(q, k, v, o, cu_seqlens, max_seq_len, workspace: torch.Tensor, block_size=128):
    """Attention stage only over the block lists (and cu_tile) held in ``workspace``."""
    lib = _lib.load()
    q, k, v, cu, T, Hq, Hk, D = _varlen_args(q, k, v, o, cu_seqlens)
    code = _dtype_code(q)
    nseq = cu.numel() - 1
    tgt = o if _tma_ok(o) else torch.empty_like(q)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    with torch.cuda.device(q.device):
        rc = lib.fpb_attention_varlen(_P(q), _P(k), _P(v), _P(tgt), code, _P(cu), nseq, T, int(max_seq_len), Hq,
                                      Hk, D, _strides(q, 2), _strides(k, 2), _strides(v, 2), _strides(tgt, 2),
                                      int(block_size), _P(workspace), workspace.numel(), _P(stream))
    _lib.check(rc)
    if tgt is not o:
        o.copy_(tgt)
    _finish(workspace, stream)


# --------------------------------------------------------------------------- paged cache
def _cuda_tensor(t, name, ndim, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got shape {tuple(t.shape)}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (flashprefill_b200 has no CPU path), got {t.device}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def _written(t, name):
    """A tensor that a kernel writes must not have two indices for one element through a stride of 0."""
    for n, s in zip(t.shape, t.stride()):
        if s == 0 and n > 1:
            raise ValueError(f"{name} is written to and must not be an expanded tensor (strides {tuple(t.stride())})")


def _cache_args(k_cache, v_cache, k_scale, v_scale, dtype, device, heads, written):
    """Checks the cache tensors; returns (cache dtype code, pages, page size, kv heads, cache strides, scale strides)."""
    _cuda_tensor(k_cache, "k_cache", 4, device)
    _cuda_tensor(v_cache, "v_cache", 4, device)
    shape, strides = k_cache.shape, k_cache.stride()
    if v_cache.shape != shape or v_cache.stride() != strides or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must share shape, strides and dtype")
    if heads is not None and shape[2] != heads:
        raise ValueError(f"the cache has {shape[2]} KV heads, expected {heads}")
    if shape[3] != 128 or strides[3] != 1:
        raise ValueError(f"the cache's last dimension must be 128 contiguous elements, got shape {tuple(shape)}, strides {strides}")
    if written:
        _written(k_cache, "k_cache")
    if k_cache.dtype is torch.float8_e4m3fn:
        if k_scale is None or v_scale is None:
            raise ValueError("an e4m3 cache needs k_scale and v_scale")
        _cuda_tensor(k_scale, "k_scale", 3, device)
        _cuda_tensor(v_scale, "v_scale", 3, device)
        if k_scale.shape != shape[:3] or v_scale.shape != shape[:3]:
            raise ValueError(f"k_scale and v_scale must have shape {tuple(shape[:3])}")
        if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
            raise TypeError("k_scale and v_scale must be float32")
        if k_scale.stride() != v_scale.stride():
            raise ValueError("k_scale and v_scale must share strides")
        if written:
            _written(k_scale, "k_scale")
        return _lib.FPB_E4M3, shape[0], shape[1], shape[2], _lib.i64arr(strides[:3]), _lib.i64arr(k_scale.stride())
    if k_cache.dtype is not dtype:
        raise TypeError(f"the cache must be {dtype} or torch.float8_e4m3fn, got {k_cache.dtype}")
    if k_scale is not None or v_scale is not None:
        raise ValueError("a 16-bit cache takes no scales")
    return _DTYPES[dtype], shape[0], shape[1], shape[2], _lib.i64arr(strides[:3]), None


def _table_args(page_table, seq_lens, batch, device):
    _cuda_tensor(page_table, "page_table", 2, device)
    _cuda_tensor(seq_lens, "seq_lens", 1, device)
    if page_table.dtype is not torch.int32 or seq_lens.dtype is not torch.int32:
        raise TypeError("page_table and seq_lens must be int32")
    if page_table.shape[0] != batch or seq_lens.shape[0] != batch:
        raise ValueError(f"page_table {tuple(page_table.shape)} and seq_lens {tuple(seq_lens.shape)} must have {batch} rows")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1 or batch > 1 and seq_lens.stride(0) != 1:
        raise ValueError("the last dimension of page_table and of seq_lens must be contiguous")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _finish_paged(stream) -> None:
    if _CHECK and not torch.cuda.is_current_stream_capturing():
        _check_paged(stream)


def _check_paged(stream) -> None:
    flags = ctypes.c_uint32(0)
    rc = _lib.load().fpb_paged_read_device_error(ctypes.byref(flags), stream)
    if rc == _lib.FPB_EDEVICE:
        what = [m for b, m in _lib.DEV_ERROR_BITS.items() if flags.value & b]
        raise _lib.FlashPrefillError("flashprefill_b200 device error: " + "; ".join(what))
    _lib.check(rc)


def check_paged_error(device=None) -> None:
    """Synchronise the current stream and raise if a paged-cache call on ``device`` (default: the current one) met a slot,
    page or length outside its tensors since the last check."""
    with torch.cuda.device(device):
        _check_paged(torch.cuda.current_stream().cuda_stream)


def kv_cache_write(k, v, k_cache, v_cache, slots, k_scale=None, v_scale=None) -> None:
    device = k.device if isinstance(k, torch.Tensor) else None
    k = _prep_input(k, "k", 3, device)
    v = _prep_input(v, "v", 3, device)
    T, Hk, D = k.shape
    if v.shape != k.shape:
        raise ValueError(f"v shape {tuple(v.shape)} must equal k shape {tuple(k.shape)}")
    if v.dtype != k.dtype:
        raise TypeError("k and v must share one dtype")
    code = _dtype_code(k)
    ccode, pages, page_size, _, cs, ss = _cache_args(k_cache, v_cache, k_scale, v_scale, k.dtype, device, Hk, True)
    _cuda_tensor(slots, "slots", 1, device)
    if slots.dtype is not torch.int64 and slots.dtype is not torch.int32:
        raise TypeError(f"slots must be int64 or int32, got {slots.dtype}")
    if slots.shape[0] != T:
        raise ValueError(f"slots must have one entry for each of the {T} rows, got {slots.shape[0]}")
    slots = slots.contiguous()
    if _CHECK and not torch.cuda.is_current_stream_capturing():
        used = slots[slots >= 0]
        if used.unique().numel() != used.numel():
            raise ValueError("two rows name one slot")
    stream = torch.cuda.current_stream(device).cuda_stream
    with torch.cuda.device(device):
        rc = _lib.load().fpb_kv_cache_write(_ptr(k), _ptr(v), code, T, Hk, D, _strides(k, 2), _strides(v, 2), _ptr(k_cache),
                                            _ptr(v_cache), ccode, pages, page_size, cs, _ptr(k_scale), _ptr(v_scale), ss,
                                            _ptr(slots), slots.element_size(), stream)
        _lib.check(rc)
        _finish_paged(stream)


def kv_cache_read(k_cache, v_cache, page_table, seq_lens, k, v, k_scale=None, v_scale=None) -> None:
    device = k_cache.device if isinstance(k_cache, torch.Tensor) else None
    for t, name in ((k, "k"), (v, "v")):
        _cuda_tensor(t, name, 4, device)
        _written(t, name)
        if not _tma_ok(t):
            raise ValueError(f"{name} must have a contiguous last dimension and 16-byte aligned rows")
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError("k and v must share shape and dtype")
    B, S, Hk, D = k.shape
    code = _dtype_code(k)
    ccode, pages, page_size, _, cs, ss = _cache_args(k_cache, v_cache, k_scale, v_scale, k.dtype, device, Hk, False)
    _table_args(page_table, seq_lens, B, device)
    if B == 0 or S == 0 or page_table.shape[1] == 0:
        return
    stream = torch.cuda.current_stream(device).cuda_stream
    with torch.cuda.device(device):
        rc = _lib.load().fpb_kv_cache_read(_ptr(k_cache), _ptr(v_cache), ccode, pages, page_size, Hk, D, cs, _ptr(k_scale),
                                           _ptr(v_scale), ss, _ptr(page_table), page_table.stride(0), page_table.shape[1],
                                           _ptr(seq_lens), B, _ptr(k), _ptr(v), code, S, _strides(k, 3), _strides(v, 3),
                                           stream)
        _lib.check(rc)
        _finish_paged(stream)


def paged_decode(q, k_cache, v_cache, page_table, seq_lens, out, lse=None, k_scale=None, v_scale=None, sm_scale=None,
                 workspace=None) -> None:
    device = q.device if isinstance(q, torch.Tensor) else None
    q = _prep_input(q, "q", 3, device)
    B, Hq, D = q.shape
    code = _dtype_code(q)
    _cuda_tensor(out, "out", 3, device)
    if out.shape != q.shape or out.dtype is not q.dtype:
        raise ValueError("out must be a tensor with q's shape, dtype and device")
    if out.stride(2) != 1:
        raise ValueError("out's last dimension must be contiguous")
    _written(out, "out")
    ccode, pages, page_size, Hk, cs, ss = _cache_args(k_cache, v_cache, k_scale, v_scale, q.dtype, device, None, False)
    if Hk == 0 or Hq % Hk:
        raise ValueError(f"num_q_heads ({Hq}) must be a multiple of num_kv_heads ({Hk})")
    _table_args(page_table, seq_lens, B, device)
    if lse is not None:
        _cuda_tensor(lse, "lse", 2, device)
        if lse.shape != q.shape[:2] or lse.dtype is not torch.float32 or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous float32 tensor of shape {(B, Hq)}")
    if B == 0 or Hq == 0:
        return
    lib = _lib.load()
    max_pages = page_table.shape[1]
    stream = torch.cuda.current_stream(device).cuda_stream
    with torch.cuda.device(device):
        if workspace is None:
            n = lib.fpb_paged_decode_workspace_bytes(B, Hq, Hk, ccode, max_pages, page_size)
            if n:
                workspace = torch.empty(n, dtype=torch.uint8, device=device)
        else:
            _cuda_tensor(workspace, "workspace", 1, device)
        rc = lib.fpb_paged_decode(_ptr(q), code, B, Hq, Hk, D, _strides(q, 2), _ptr(k_cache), _ptr(v_cache), ccode, pages,
                                  page_size, cs, _ptr(k_scale), _ptr(v_scale), ss, _ptr(page_table), page_table.stride(0),
                                  max_pages, _ptr(seq_lens), _ptr(out), _strides(out, 2), _ptr(lse),
                                  1.0 / 128 ** 0.5 if sm_scale is None else float(sm_scale), _ptr(workspace),
                                  0 if workspace is None else workspace.numel() * workspace.element_size(), stream)
        _lib.check(rc)
        _finish_paged(stream)


def paged_decode_workspace_bytes(batch, q_heads, kv_heads, cache_dtype, max_pages, page_size) -> int:
    """Bytes of workspace that paged_decode needs for these sizes."""
    code = _lib.FPB_E4M3 if cache_dtype is torch.float8_e4m3fn else _DTYPES[cache_dtype]
    return _lib.load().fpb_paged_decode_workspace_bytes(batch, q_heads, kv_heads, code, max_pages, page_size)
