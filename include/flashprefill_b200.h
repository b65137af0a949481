/* flashprefill_b200 -- C ABI of the B200 (sm_100a) sparse-prefill operator.
 *
 * The library replaces the device work behind the two public entry points of
 * FlashPrefill (qhfan/FlashPrefill, paths relative to that project):
 *   ops/flashprefill_native_forward.py:481-499  flash_prefill(q, k, v, out, block_size,
 *       attention_sink, window_size, alpha, last_n_block_full, min_budget)
 *   ops/flashprefill_varlen_func.py:723-743     flash_prefill_varlen_func(q, k, v, o,
 *       cu_seqlens, max_seq_len, alpha, block_size, attention_sink, window_size, last_n_block)
 * Those Python functions launch Triton kernels; here the same work is three CUDA kernels
 * (pooled keys, fused block search, tcgen05 block-sparse attention).  All pointers are
 * device pointers unless stated; all calls are asynchronous on `stream` (a cudaStream_t,
 * NULL = legacy default stream) and never synchronise the host, except
 * fpb_read_device_error.  Return value: FPB_OK or an FPB_E* code; fpb_last_error()
 * describes the most recent failure of the calling thread.
 *
 * Tensor layout: dense q/k/v/out are (batch, seq, heads, 128) with the last dimension
 * contiguous and strides given in ELEMENTS as {batch, seq, head}; varlen tensors are
 * (tokens, heads, 128) with strides {token, head}.  Strides must be multiples of 8
 * elements (16 bytes) and base pointers 16-byte aligned.  dtype: FPB_BF16 or FPB_FP16;
 * q, k, v and out share it.  head_dim and block_size must be 128.
 *
 * Workspace: the caller provides `workspace` of at least the size returned by the
 * matching *_workspace_bytes function (the reference allocates its temporaries from the
 * PyTorch caching allocator, native:419-434 / varlen:596-663; here they are one caller
 * buffer).  It holds the device error word, cu_tile, the pooled keys, and the per-head
 * block lists.  Its layout is reported by fpb_workspace_layout.
 */
#ifndef FLASHPREFILL_B200_H
#define FLASHPREFILL_B200_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define FPB_API __attribute__((visibility("default")))
#else
#define FPB_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define FPB_OK 0
#define FPB_EINVAL 1   /* invalid argument (shape, dtype, stride, alignment, size) */
#define FPB_ECUDA 2    /* a CUDA runtime/driver call or a kernel launch failed */
#define FPB_EDEVICE 3  /* fpb_read_device_error found error bits set */

#define FPB_BF16 0
#define FPB_FP16 1
#define FPB_E4M3 2 /* paged caches only: 8-bit codes with a float scale for each (token, head) */

/* Device error bits (fpb_read_device_error). */
#define FPB_DEV_WAIT_TIMEOUT 1u   /* a pipeline wait ran out of time; the kernel bailed out */
#define FPB_DEV_BAD_SEQLENS 2u    /* cu_seqlens not non-decreasing from 0 to total_tokens */
#define FPB_DEV_SEQ_TOO_LONG 4u   /* a sequence longer than max_seq_len (rows skipped) */
#define FPB_DEV_INDEX_RANGE 8u    /* a block list held an index outside [0, query block] */
#define FPB_DEV_BAD_PAGE 16u      /* paged cache: a slot or page-table entry outside the cache (skipped) */
#define FPB_DEV_BAD_LENGTH 32u    /* paged cache: a sequence length outside [0, room] */

/* Library version (major*10000 + minor*100 + patch). */
FPB_API int fpb_version(void);

/* Message for the last failing call on this thread ("" if none). */
FPB_API const char* fpb_last_error(void);

/* Workspace size for the dense entry points (replaces the temporaries of
 * ops/flashprefill_native_forward.py:419-434 and deal_output_score's outputs :379-385). */
FPB_API size_t fpb_dense_workspace_bytes(int batch, int seqlen, int hq, int hk, int head_dim);

/* Workspace size for the varlen entry points (replaces
 * ops/flashprefill_varlen_func.py:596-698).  Sized from host-known bounds only, so no
 * device->host copy of cu_seqlens is needed. */
FPB_API size_t fpb_varlen_workspace_bytes(int total_tokens, int nseq, int max_seq_len, int hq, int hk,
                                          int head_dim);

/* Byte offsets inside the workspace.  out[8] = {error word, cu_tile (int32[nseq+1]),
 * pooled keys (dtype[tiles][hk][128]), counts (int32[hq][tiles]), block lists
 * (int32[hq][tiles][cap]), total bytes, tiles, cap}.  Row `tile_base(seq)+qb` of head h:
 * counts[h*tiles + row] entries at lists[(h*tiles + row)*cap ...], ascending.
 * varlen = 0: a = batch, b = seqlen, c ignored.  varlen = 1: a = nseq, b = total_tokens,
 * c = max_seq_len.  (The reference keeps the same information as block_index/counts,
 * native:377-385, or out_index/out_number_cu, varlen:683-698.) */
FPB_API int fpb_workspace_layout(int varlen, int a, int b, int c, int hq, int hk, int head_dim, int64_t* out8);

/* Whole operator, dense layout: replaces FlashPrefill.forward
 * (ops/flashprefill_native_forward.py:405-476).  Writes out in place.
 * mean_model: 4 or 8, the warp count whose reduction order the pooled-key sum follows
 * (the reference autotunes it, native:7-20). */
FPB_API int fpb_prefill_dense(const void* q, const void* k, const void* v, void* out, int dtype, int batch,
                              int seqlen, int hq, int hk, int head_dim, const int64_t* q_strides,
                              const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                              int block_size, int attention_sink, int window_size, float alpha,
                              int last_n_block_full, int min_budget, int mean_model, void* workspace,
                              size_t workspace_bytes, void* stream);

/* Whole operator, packed varlen layout: replaces FlashPrefill_varlen.forward
 * (ops/flashprefill_varlen_func.py:577-720).  cu_seqlens: device int32[nseq+1]. */
FPB_API int fpb_prefill_varlen(const void* q, const void* k, const void* v, void* o, int dtype,
                               const int32_t* cu_seqlens, int nseq, int total_tokens, int max_seq_len, int hq,
                               int hk, int head_dim, const int64_t* q_strides, const int64_t* k_strides,
                               const int64_t* v_strides, const int64_t* o_strides, int block_size,
                               int attention_sink, int window_size, float alpha, int last_n_block, int mean_model,
                               void* workspace, size_t workspace_bytes, void* stream);

/* fpb_prefill_dense for one rank of a head-sharded layer that also needs the full output on
 * every GPU (the gather of head shards; the reference has no multi-GPU path of its own).
 * `out` is this rank's head slice of its full (B, S, Hq, D) output; out_peers[i] is the
 * address of the same slice in another GPU's copy of that output (identical layout and
 * strides), reachable from this GPU (peer access or a symmetric-memory mapping).  The
 * attention epilogue writes every output tile to `out` and, with 16-byte stores over
 * NVLink, to each peer, so the gather overlaps the attention.  The call returns when the
 * work is queued: the caller orders the peers' reads after every rank's kernel (a
 * cross-GPU barrier on the stream).  n_peers <= 7. */
FPB_API int fpb_prefill_dense_peers(const void* q, const void* k, const void* v, void* out, int dtype, int batch,
                                    int seqlen, int hq, int hk, int head_dim, const int64_t* q_strides,
                                    const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                                    int block_size, int attention_sink, int window_size, float alpha,
                                    int last_n_block_full, int min_budget, int mean_model, void* workspace,
                                    size_t workspace_bytes, void* const* out_peers, int n_peers, void* stream);

/* fpb_prefill_dense restricted to the query blocks [q_block_begin, q_block_end) of every batch
 * entry: their block lists are searched and their output rows written, with the selection
 * rules of the whole sequence (the last-N rule still refers to the sequence's last blocks);
 * other output rows are left untouched.  The union over a partition of [0, ceil(S/128)) of
 * such calls equals one fpb_prefill_dense call.  It serves a 2-D split of one layer over
 * GPUs (KV-head groups x query-block ranges, each GPU holding its heads' whole K/V) when
 * there are more GPUs than KV heads.  The reference runs whole layers only
 * (ops/flashprefill_native_forward.py:481-499); q/k/v/out and the workspace are as in
 * fpb_prefill_dense. */
FPB_API int fpb_prefill_dense_rows(const void* q, const void* k, const void* v, void* out, int dtype, int batch,
                                   int seqlen, int hq, int hk, int head_dim, const int64_t* q_strides,
                                   const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                                   int block_size, int attention_sink, int window_size, float alpha,
                                   int last_n_block_full, int min_budget, int mean_model, int q_block_begin,
                                   int q_block_end, void* workspace, size_t workspace_bytes, void* stream);

/* Chunked (prefix) prefill: the queries are the last q_len positions of a kv_len-token sequence
 * (q and out (B, q_len, Hq, D); k and v (B, kv_len, Hk, D), the cached prefix followed by the
 * chunk).  Block structure, pooled keys and the selection rules are those of the whole
 * kv_len-token sequence (the last-N rule refers to its last blocks); a query block that starts
 * before the chunk scores its missing rows as zero rows, as the search scores the padded rows of
 * a partial last block.  The workspace is that of fpb_prefill_dense for kv_len tokens.  With
 * q_len = kv_len it equals fpb_prefill_dense.  No counterpart in the reference, which sends
 * chunked prefills to dense attention (patches/patch_loader_vllm_0_10_0.py:272-300,
 * ruler/models/llama.py:310-333). */
FPB_API int fpb_prefill_dense_chunk(const void* q, const void* k, const void* v, void* out, int dtype, int batch,
                                    int q_len, int kv_len, int hq, int hk, int head_dim, const int64_t* q_strides,
                                    const int64_t* k_strides, const int64_t* v_strides,
                                    const int64_t* o_strides, int block_size, int attention_sink,
                                    int window_size, float alpha, int last_n_block_full, int min_budget,
                                    int mean_model, void* workspace, size_t workspace_bytes, void* stream);

/* Search stage only (pooled keys + block lists into the workspace): replaces
 * compute_mean_vector + compute_block_score + normalize_scores + deal_output_score
 * (ops/flashprefill_native_forward.py:22-188,347-403). */
FPB_API int fpb_search_dense(const void* q, const void* k, int dtype, int batch, int seqlen, int hq, int hk,
                             int head_dim, const int64_t* q_strides, const int64_t* k_strides, int block_size,
                             int attention_sink, int window_size, float alpha, int last_n_block_full,
                             int min_budget, int mean_model, void* workspace, size_t workspace_bytes, void* stream);

/* Search stage only, varlen: replaces ops/flashprefill_varlen_func.py:8-18,35-409,656-698. */
FPB_API int fpb_search_varlen(const void* q, const void* k, int dtype, const int32_t* cu_seqlens, int nseq,
                              int total_tokens, int max_seq_len, int hq, int hk, int head_dim,
                              const int64_t* q_strides, const int64_t* k_strides, int block_size,
                              int attention_sink, int window_size, float alpha, int last_n_block, int mean_model,
                              void* workspace, size_t workspace_bytes, void* stream);

/* Attention stage only, over the block lists already in the workspace (written by
 * fpb_search_* or by the caller): replaces _flash_forward
 * (ops/flashprefill_native_forward.py:228-344). */
FPB_API int fpb_attention_dense(const void* q, const void* k, const void* v, void* out, int dtype, int batch,
                                int seqlen, int hq, int hk, int head_dim, const int64_t* q_strides,
                                const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                                int block_size, void* workspace, size_t workspace_bytes, void* stream);

/* Attention stage only, varlen: replaces _flash_block_sparse_varlen
 * (ops/flashprefill_varlen_func.py:449-575).  Needs cu_tile in the workspace, which
 * fpb_search_varlen writes. */
FPB_API int fpb_attention_varlen(const void* q, const void* k, const void* v, void* o, int dtype,
                                 const int32_t* cu_seqlens, int nseq, int total_tokens, int max_seq_len, int hq,
                                 int hk, int head_dim, const int64_t* q_strides, const int64_t* k_strides,
                                 const int64_t* v_strides, const int64_t* o_strides, int block_size,
                                 void* workspace, size_t workspace_bytes, void* stream);

/* Dense prefill that allocates nothing, for callers that cannot call cudaMalloc or pass
 * a workspace (runtimes that forbid allocation on their hot path, hosts without a device
 * allocator).  No counterpart in the reference.  Same arguments and results as
 * fpb_prefill_dense without the workspace: it uses a 32 MiB device array inside the
 * library, held by every GPU that loads the library until exit.  Problems whose required
 * workspace (the error word, pooled keys, counts and block lists: every part of
 * fpb_dense_workspace_bytes except the optional long-row split area) exceeds 32 MiB are
 * rejected with FPB_EINVAL (e.g. 32K tokens with 32/8 heads fit; 128K do not); long rows
 * are split only when the split area fits in the array as well.  The first call on a
 * device looks up the array's address on that device and should come before any stream
 * capture.  Calls share the array: calls that overlap on the GPU race.  Device-side errors
 * of these calls are read with fpb_noalloc_read_device_error. */
FPB_API int fpb_prefill_dense_noalloc(const void* q, const void* k, const void* v, void* out, int dtype, int batch,
                                      int seqlen, int hq, int hk, int head_dim, const int64_t* q_strides,
                                      const int64_t* k_strides, const int64_t* v_strides,
                                      const int64_t* o_strides, int block_size, int attention_sink,
                                      int window_size, float alpha, int last_n_block_full, int min_budget,
                                      int mean_model, void* stream);

/* fpb_read_device_error for the no-allocation path: synchronises `stream` and reads the
 * error word of the current device's fixed scratch array (the last
 * fpb_prefill_dense_noalloc call on that device).  No counterpart in the reference. */
FPB_API int fpb_noalloc_read_device_error(uint32_t* flags, void* stream);

/* Test hook, no counterpart in the reference: on the current device, sets the limit of every
 * bounded device-side wait (default 1 s; accepted range 1 ms .. 1 s) and, when
 * withhold_first_load is non-zero, arms a one-shot fault: the next attention launch on the
 * device skips one key-tile load (the first producer to reach one consumes the fault), so
 * that one of its waits runs out and the call reports FPB_DEV_WAIT_TIMEOUT through the
 * error word.  Call it again with (0, 1000000000) to restore normal operation.  For tests
 * of the timeout path only. */
FPB_API int fpb_test_set_fault(int withhold_first_load, unsigned long long wait_limit_ns);

/* Synchronises `stream`, copies the device error word of `workspace` to *flags and
 * returns FPB_EDEVICE if any bit is set.  No counterpart in the reference, which has no
 * device-side error reporting. */
FPB_API int fpb_read_device_error(const void* workspace, uint32_t* flags, void* stream);

/* ---- Paged key/value cache and decode attention (no counterpart in the reference, which leaves decode to its host
 * framework).  A cache is (num_pages, page_size, hk, 128): k_cache and v_cache share cache_strides = {page, token, head}
 * in ELEMENTS (multiples of 16 bytes; last dimension contiguous).  cache_dtype is the rows' dtype, or FPB_E4M3: codes with
 * k_scale / v_scale, float (num_pages, page_size, hk) with scale_strides = {page, token, head} in elements; a value is
 * code * scale.  16-bit caches take NULL scales.  page_table: int32 (batch, max_pages), row stride table_stride;
 * seq_lens: int32 (batch).  Both live on the device and are checked there: an entry that points outside the cache, a slot
 * beyond it or a length outside [0, room] sets an error bit of the current device, which stays until
 * fpb_paged_read_device_error reads it; nothing outside the tensors is touched. */

/* Rows k, v (tokens, hk, 128), strides {token, head}, into the cache slots slots[t] = page * page_size + offset (int32 or
 * int64: slot_bytes 4 or 8).  A negative slot skips its row (padding).  Slots must differ from one another; where two rows
 * name one slot, what it holds is not defined.  k_cache and v_cache are different memory, as are k_scale and v_scale.  For
 * FPB_E4M3 each row's scale is max(max|x|, 2^-100) / 448. */
FPB_API int fpb_kv_cache_write(const void* k, const void* v, int dtype, int tokens, int hk, int head_dim,
                               const int64_t* k_strides, const int64_t* v_strides, void* k_cache, void* v_cache,
                               int cache_dtype, int num_pages, int page_size, const int64_t* cache_strides,
                               float* k_scale, float* v_scale, const int64_t* scale_strides, const void* slots,
                               int slot_bytes, void* stream);

/* The first seq_lens[b] cached rows of every sequence into k, v (batch, out_len, hk, 128), strides {batch, token, head}.
 * Later rows, and those of a sequence or page that is in error, are left as they were. */
FPB_API int fpb_kv_cache_read(const void* k_cache, const void* v_cache, int cache_dtype, int num_pages, int page_size,
                              int hk, int head_dim, const int64_t* cache_strides, const float* k_scale,
                              const float* v_scale, const int64_t* scale_strides, const int32_t* page_table,
                              int64_t table_stride, int max_pages, const int32_t* seq_lens, int batch, void* k, void* v,
                              int dtype, int out_len, const int64_t* k_strides, const int64_t* v_strides, void* stream);

/* Workspace of fpb_paged_decode.  It follows from the batch, the heads and the table's width, max_pages * page_size (not from the
 * lengths), and is 0 where sequences of that width are short enough to be joined in shared memory. */
FPB_API size_t fpb_paged_decode_workspace_bytes(int batch, int hq, int hk, int cache_dtype, int max_pages,
                                                int page_size);

/* Attention of one new token a sequence, q (batch, hq, 128), over its seq_lens[b] cached tokens (the new token's own row
 * is written first, by fpb_kv_cache_write).  out like q, strides {batch, head}; lse: NULL or float (batch, hq) contiguous,
 * the natural logarithm of the sum of exp(sm_scale q.k).  A sequence of length 0 (or in error) gives zeros and -inf; tokens
 * of a page in error are left out.  The workspace needs no initialisation; calls that overlap on the GPU need one each. */
FPB_API int fpb_paged_decode(const void* q, int dtype, int batch, int hq, int hk, int head_dim, const int64_t* q_strides,
                             const void* k_cache, const void* v_cache, int cache_dtype, int num_pages, int page_size,
                             const int64_t* cache_strides, const float* k_scale, const float* v_scale,
                             const int64_t* scale_strides, const int32_t* page_table, int64_t table_stride,
                             int max_pages, const int32_t* seq_lens, void* out, const int64_t* o_strides, float* lse,
                             float sm_scale, void* workspace, size_t workspace_bytes, void* stream);

/* Synchronises `stream`, reads and clears the current device's paged error bits into *flags; FPB_EDEVICE if any was set. */
FPB_API int fpb_paged_read_device_error(uint32_t* flags, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FLASHPREFILL_B200_H */
