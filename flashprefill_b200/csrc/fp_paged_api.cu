// C ABI of the paged cache (fp_paged.cu) and of decode attention over it (fp_decode.cu).  Included at the end of fp_api.cu
// (one translation unit): argument checks and launches.
namespace fpb {
namespace {

FastDiv make_div(int d) {
  int log2 = 0;
  while ((int64_t(1) << log2) < d) ++log2;
  return {(unsigned)((uint64_t(1) << (31 + log2)) / d + 1), 31 + log2};
}

// Strides in units of `unit`; each must be below 2^32 units.
int make_pitch(Pitch* p, int64_t outer, int64_t tok, int64_t head, int unit, const char* what) {
  for (const int64_t s : {outer, tok, head})
    FPB_CHECK_ARG(s / unit < (int64_t(1) << 32), "%s stride of %lld %s is too large", what, (long long)s, unit > 1 ? "bytes" : "elements");
  *p = {(unsigned)(outer / unit), (unsigned)(tok / unit), (unsigned)(head / unit)};
  return FPB_OK;
}

// The cache arguments shared by the three entry points.  out: C with byte strides.
int make_cache(PagedCache* C, const void* k_cache, const void* v_cache, int cache_dtype, int dtype, int num_pages,
               int page_size, int hk, int head_dim, const int64_t* cs, const float* k_scale, const float* v_scale,
               const int64_t* ss) {
  FPB_CHECK_ARG(dtype == FPB_BF16 || dtype == FPB_FP16, "dtype must be FPB_BF16 or FPB_FP16 (got %d)", dtype);
  FPB_CHECK_ARG(cache_dtype == dtype || cache_dtype == FPB_E4M3,
                "the cache must hold the rows' 16-bit type or FPB_E4M3 (got %d for rows of %d)", cache_dtype, dtype);
  FPB_CHECK_ARG(head_dim == kHeadDim, "head_dim must be 128 (got %d)", head_dim);
  FPB_CHECK_ARG(num_pages >= 1 && page_size >= 1 && hk >= 1, "num_pages (%d), page_size (%d) and num_kv_heads (%d) must be >= 1",
                num_pages, page_size, hk);
  FPB_TRY(check_ptr(k_cache, "k_cache"));
  FPB_TRY(check_ptr(v_cache, "v_cache"));
  const int elt = cache_dtype == FPB_E4M3 ? 1 : 2;
  FPB_CHECK_ARG(cs != nullptr, "cache strides are NULL");
  for (int i = 0; i < 3; ++i) {
    FPB_CHECK_ARG(cs[i] >= 0 && cs[i] * elt % 16 == 0, "cache stride[%d]=%lld must be a non-negative multiple of 16 bytes", i,
                  (long long)cs[i]);
  }
  C->k = static_cast<uint8_t*>(const_cast<void*>(k_cache));
  C->v = static_cast<uint8_t*>(const_cast<void*>(v_cache));
  FPB_TRY(make_pitch(&C->rows, cs[0] * elt, cs[1] * elt, cs[2] * elt, 16, "cache"));
  C->num_pages = num_pages;
  C->page_size = page_size;
  C->page_of = make_div(page_size);
  C->k_scale = C->v_scale = nullptr;
  C->scales = Pitch{0, 0, 0};
  if (cache_dtype == FPB_E4M3) {
    FPB_CHECK_ARG(k_scale != nullptr && v_scale != nullptr, "an e4m3 cache needs k_scale and v_scale");
    FPB_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) & 3) == 0,
                  "k_scale and v_scale must be aligned float pointers");
    FPB_CHECK_ARG(ss != nullptr, "scale strides are NULL");
    for (int i = 0; i < 3; ++i) FPB_CHECK_ARG(ss[i] >= 0, "scale stride[%d]=%lld is negative", i, (long long)ss[i]);
    FPB_TRY(make_pitch(&C->scales, ss[0], ss[1], ss[2], 1, "scale"));
    C->k_scale = const_cast<float*>(k_scale);
    C->v_scale = const_cast<float*>(v_scale);
  } else {
    FPB_CHECK_ARG(k_scale == nullptr && v_scale == nullptr, "a 16-bit cache takes no scales");
  }
  return FPB_OK;
}

int check_table(const int32_t* table, int64_t stride, int max_pages, int page_size, const int32_t* seq_lens, int batch) {
  FPB_CHECK_ARG(batch >= 1 && max_pages >= 1, "batch (%d) and max_pages (%d) must be >= 1", batch, max_pages);
  FPB_CHECK_ARG((int64_t)max_pages * page_size <= kPagedMaxLen, "max_pages * page_size must be at most %lld",
                (long long)kPagedMaxLen);
  FPB_CHECK_ARG(table != nullptr && (reinterpret_cast<uintptr_t>(table) & 3) == 0, "page_table must be an aligned int32 pointer");
  FPB_CHECK_ARG(seq_lens != nullptr && (reinterpret_cast<uintptr_t>(seq_lens) & 3) == 0,
                "seq_lens must be an aligned int32 pointer");
  FPB_CHECK_ARG(stride >= 0 && stride < (int64_t(1) << 40), "page_table stride %lld is out of range", (long long)stride);
  return FPB_OK;
}

// Launches a kernel that begins with await_stream(), in clusters of `cluster` CTAs.
template <typename... P, typename... V>
int launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream, const V&... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attrs[2] = {};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  FPB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  return FPB_OK;
}

// Launches a read kernel with one token of a head for 16 lanes, or with kReadGroup where page_size allows it and every SM
// still gets the 8 blocks it holds.
constexpr int kReadGroup = 4;
template <typename T, bool kE4m3>
int launch_read(const KvReadArgs& A, int batch, cudaStream_t stream) {
  constexpr int kBlock = block_rows(false);
  const bool grouped = A.C.page_size % kReadGroup == 0 && (int64_t)A.out_len * A.hk * batch >= (int64_t)kReadGroup * kBlock * 148 * 8;
  const unsigned per = grouped ? kReadGroup : 1, items = ((unsigned)A.out_len + per - 1) / per * (unsigned)A.hk;
  const dim3 grid((items + kBlock - 1) / kBlock, batch);
  return launch(grouped ? kv_read_kernel<T, kE4m3, kReadGroup> : kv_read_kernel<T, kE4m3, 1>, grid, kRowThreads, 0, 1, stream, A);
}

// How the query heads of a KV head become items: equal groups of at most 16.
void head_groups(int G, int* ngroups, int* nh) {
  const int n = (G + 15) / 16;
  *nh = (G + n - 1) / n;
  *ngroups = (G + *nh - 1) / *nh;
}

// How a call runs.  Every size here is a bound from the table's width: lengths are known on the device only.
//
// Short sequences: a cluster for each item, if no warp gets more than kShortTiles tiles that way: as many CTAs as the GPU holds
// at once, 8 at most; wide CTAs where a warp's tiles, one after another, are fewer that way (32/8 heads, bf16: 1 x 4096 tokens
// 10.6 us with 8 x 4 warps an item, 7.7 with 8 x 12; 1 x 500, one tile a warp either way, 4.5 and 6.0).
// Else pieces of the line of all units.  Clusters win up to there (1 x 8192 tokens 10.6 us, 13.0 in pieces; 256 x up to 600 of
// 8/2 heads 18.3 and 21.4; 64 x up to 1024, 16 tiles, 27.6 and 28.2) and lose beyond (32 x up to 2100, 33 tiles, 41 us and 29.3
// in pieces; 8 x up to 32000 of 48/4 heads, e4m3 to bf16, 54 and 41).  Few items, each of several pieces, take wide CTAs, which leave a
// third as many partial sums (2 x up to 262144 tokens of 28/4 heads, e4m3: 81.6 us, narrow 82.5); many ragged ones narrow CTAs,
// which wait for one another less (64 x up to 8192 of 32/8: 168 us, wide 172).
constexpr int kSms = 148;
constexpr int kShortTiles = 16;
struct DecodeShape {
  int G, ngroups, nh;
  int warps, cluster;    // of a CTA; cluster 0: pieces
  int pieces;            // CTAs: the places of a 148-SM GPU
  int by_item, join_heads;
  int64_t items, units;  // all items; all units at most
};
DecodeShape decode_shape(int batch, int hq, int hk, int cache_dtype, int max_pages, int page_size) {
  DecodeShape s{};
  s.G = hq / hk;
  head_groups(s.G, &s.ngroups, &s.nh);
  const int nt = s.nh <= 8 ? 1 : 2, tile = cache_dtype == FPB_E4M3 ? 32 : 16;
  const int64_t tiles = ((int64_t)max_pages * page_size + tile - 1) / tile;
  s.items = (int64_t)batch * hk * s.ngroups;
  // the largest cluster of CTAs of `warps` warps that fits with all others, and the tiles of a warp
  auto cluster = [&](int warps) {
    const int64_t units = (tiles + warps - 1) / warps, places = kSms * dec_ctas_per_sm(nt, warps);
    int c = 1;
    while (c < kDecMaxCluster && 2 * c <= units && s.items * 2 * c <= places) c *= 2;
    return c;
  };
  auto each_warp = [&](int warps) { return (tiles + warps * cluster(warps) - 1) / (warps * cluster(warps)); };
  const int wide = wide_warps(nt);
  s.warps = s.items <= kSms && each_warp(wide) < each_warp(kNarrow) ? wide : kNarrow;
  s.cluster = cluster(s.warps);
  if (each_warp(s.warps) > kShortTiles || s.items * s.cluster >= (int64_t(1) << 31)) {
    s.cluster = 0;
    s.warps = 2 * s.items <= kSms ? wide : kNarrow;
  }
  s.units = s.items * ((tiles + s.warps - 1) / s.warps + 1);
  s.pieces = (int)std::min<int64_t>(kSms * dec_ctas_per_sm(nt, s.warps), s.units);
  s.by_item = s.items <= s.pieces;
  // an item of many pieces has a CTA of the join for each head (2 x up to 262144 tokens of 28/4 heads, e4m3: 81.6 us, 85.4 without)
  s.join_heads = s.pieces / s.items >= 16 ? 1 : std::min(s.nh, kJoinThreads / 32);
  return s;
}
int decode_descs(const DecodeShape& s) { return s.by_item ? (int)s.items : s.pieces; }
int64_t decode_ws_part(const DecodeShape& s) { return align256(16 * (int64_t)decode_descs(s)); }
int64_t decode_ws_ml(const DecodeShape& s) {
  return decode_ws_part(s) + align256(2 * (int64_t)s.pieces * s.nh * kHeadDim * 4);
}
int64_t decode_ws_total(const DecodeShape& s) {
  return s.cluster ? 0 : decode_ws_ml(s) + align256(2 * (int64_t)s.pieces * s.nh * 8);
}

template <typename T, bool kE4m3, int NT>
int launch_decode(const DecodeArgs& A, const DecodeShape& s, cudaStream_t stream) {
  const int smem = dec_smem_bytes(s.warps);
  if (s.cluster) {
    auto kernel = s.warps == kNarrow ? paged_decode_short_kernel<T, kE4m3, NT, kNarrow>
                                     : paged_decode_short_kernel<T, kE4m3, NT, wide_warps(NT)>;
    FPB_TRY(set_smem(kernel, smem));
    return launch(kernel, dim3((unsigned)(s.items * s.cluster)), s.warps * 32, smem, s.cluster, stream, A, s.cluster);
  }
  auto kernel = s.warps == kNarrow ? paged_decode_kernel<T, kE4m3, NT, kNarrow> : paged_decode_kernel<T, kE4m3, NT, wide_warps(NT)>;
  FPB_TRY(set_smem(kernel, smem));
  FPB_TRY(launch(kernel, dim3(s.pieces), s.warps * 32, smem, 1, stream, A));
  return launch(paged_decode_join_kernel<T>, dim3(decode_descs(s), (s.nh + s.join_heads - 1) / s.join_heads), kJoinThreads, 0, 1,
                stream, A);
}

}  // namespace
}  // namespace fpb

extern "C" {

int fpb_kv_cache_write(const void* k, const void* v, int dtype, int tokens, int hk, int head_dim, const int64_t* k_strides,
                       const int64_t* v_strides, void* k_cache, void* v_cache, int cache_dtype, int num_pages, int page_size,
                       const int64_t* cache_strides, float* k_scale, float* v_scale, const int64_t* scale_strides,
                       const void* slots, int slot_bytes, void* stream) {
  KvWriteArgs A{};
  FPB_TRY(make_cache(&A.C, k_cache, v_cache, cache_dtype, dtype, num_pages, page_size, hk, head_dim, cache_strides, k_scale,
                     v_scale, scale_strides));
  FPB_CHECK_ARG(tokens >= 0, "tokens (%d) must be >= 0", tokens);
  FPB_CHECK_ARG((int64_t)tokens * hk < (int64_t(1) << 31) - 32, "tokens * num_kv_heads must be below 2^31");
  FPB_CHECK_ARG(slot_bytes == 4 || slot_bytes == 8, "slot_bytes must be 4 or 8 (got %d)", slot_bytes);
  if (tokens == 0) return FPB_OK;
  FPB_TRY(check_ptr(k, "k"));
  FPB_TRY(check_ptr(v, "v"));
  FPB_TRY(check_strides(k_strides, 2, "k"));
  FPB_TRY(check_strides(v_strides, 2, "v"));
  FPB_CHECK_ARG(slots != nullptr && reinterpret_cast<uintptr_t>(slots) % slot_bytes == 0, "slots must be an aligned pointer");
  FPB_CHECK_ARG(k_cache != v_cache, "k_cache and v_cache must not be the same memory");
  FPB_CHECK_ARG(k_scale == nullptr || k_scale != v_scale, "k_scale and v_scale must not be the same memory");
  A.k = static_cast<const uint8_t*>(k);
  A.v = static_cast<const uint8_t*>(v);
  FPB_TRY(make_pitch(&A.kp, 0, 2 * k_strides[0], 2 * k_strides[1], 16, "k"));
  FPB_TRY(make_pitch(&A.vp, 0, 2 * v_strides[0], 2 * v_strides[1], 16, "v"));
  A.token_of = make_div(hk);
  A.slots = slots;
  A.slots64 = slot_bytes == 8;
  A.rows = (unsigned)tokens * (unsigned)hk;
  A.hk = hk;
  auto st = static_cast<cudaStream_t>(stream);
  const unsigned per = block_rows(cache_dtype == FPB_E4M3), blocks = (A.rows + per - 1) / per;
  return launch(cache_dtype != FPB_E4M3 ? kv_write_kernel<__half, false>
                : dtype == FPB_BF16     ? kv_write_kernel<__nv_bfloat16, true>
                                        : kv_write_kernel<__half, true>,
                dim3(blocks), kRowThreads, 0, 1, st, A);
}

int fpb_kv_cache_read(const void* k_cache, const void* v_cache, int cache_dtype, int num_pages, int page_size, int hk,
                      int head_dim, const int64_t* cache_strides, const float* k_scale, const float* v_scale,
                      const int64_t* scale_strides, const int32_t* page_table, int64_t table_stride, int max_pages,
                      const int32_t* seq_lens, int batch, void* k, void* v, int dtype, int out_len, const int64_t* k_strides,
                      const int64_t* v_strides, void* stream) {
  KvReadArgs A{};
  FPB_TRY(make_cache(&A.C, k_cache, v_cache, cache_dtype, dtype, num_pages, page_size, hk, head_dim, cache_strides, k_scale,
                     v_scale, scale_strides));
  FPB_TRY(check_table(page_table, table_stride, max_pages, page_size, seq_lens, batch));
  FPB_CHECK_ARG(batch <= 65535, "batch (%d) must be at most 65535", batch);
  FPB_CHECK_ARG(out_len >= 1 && ((int64_t)out_len + 3) * hk < (int64_t(1) << 31) - 16,
                "out_len (%d) must be >= 1 and out_len * num_kv_heads below 2^31", out_len);
  FPB_TRY(check_ptr(k, "k"));
  FPB_TRY(check_ptr(v, "v"));
  FPB_TRY(check_strides(k_strides, 3, "k"));
  FPB_TRY(check_strides(v_strides, 3, "v"));
  FPB_CHECK_ARG(k != v, "k and v must not be the same memory");
  A.page_table = page_table;
  A.table_stride = table_stride;
  A.max_pages = max_pages;
  A.seq_lens = seq_lens;
  A.out_len = out_len;
  A.hk = hk;
  A.k = static_cast<uint8_t*>(k);
  A.v = static_cast<uint8_t*>(v);
  FPB_TRY(make_pitch(&A.kp, 2 * k_strides[0], 2 * k_strides[1], 2 * k_strides[2], 16, "k"));
  FPB_TRY(make_pitch(&A.vp, 2 * v_strides[0], 2 * v_strides[1], 2 * v_strides[2], 16, "v"));
  A.group_of = make_div(hk);
  auto st = static_cast<cudaStream_t>(stream);
  if (cache_dtype != FPB_E4M3) return launch_read<__half, false>(A, batch, st);
  return dtype == FPB_BF16 ? launch_read<__nv_bfloat16, true>(A, batch, st) : launch_read<__half, true>(A, batch, st);
}

size_t fpb_paged_decode_workspace_bytes(int batch, int hq, int hk, int cache_dtype, int max_pages, int page_size) {
  if (batch < 1 || hq < 1 || hk < 1 || hq % hk != 0 || max_pages < 1 || page_size < 1) return 0;
  return (size_t)decode_ws_total(decode_shape(batch, hq, hk, cache_dtype, max_pages, page_size));
}

int fpb_paged_decode(const void* q, int dtype, int batch, int hq, int hk, int head_dim, const int64_t* q_strides,
                     const void* k_cache, const void* v_cache, int cache_dtype, int num_pages, int page_size,
                     const int64_t* cache_strides, const float* k_scale, const float* v_scale, const int64_t* scale_strides,
                     const int32_t* page_table, int64_t table_stride, int max_pages, const int32_t* seq_lens, void* out,
                     const int64_t* o_strides, float* lse, float sm_scale, void* workspace, size_t workspace_bytes,
                     void* stream) {
  DecodeArgs A{};
  FPB_TRY(make_cache(&A.C, k_cache, v_cache, cache_dtype, dtype, num_pages, page_size, hk, head_dim, cache_strides, k_scale,
                     v_scale, scale_strides));
  FPB_CHECK_ARG(hq >= 1 && hq % hk == 0, "num_q_heads (%d) must be a multiple of num_kv_heads (%d)", hq, hk);
  FPB_TRY(check_table(page_table, table_stride, max_pages, page_size, seq_lens, batch));
  FPB_CHECK_ARG((int64_t)batch * hq < (int64_t(1) << 31), "batch * num_q_heads must be below 2^31");
  FPB_TRY(check_ptr(q, "q"));
  FPB_TRY(check_strides(q_strides, 2, "q"));
  FPB_CHECK_ARG(out != nullptr && (reinterpret_cast<uintptr_t>(out) & 1) == 0, "out must be an aligned pointer");
  FPB_CHECK_ARG(o_strides != nullptr, "out strides are NULL");
  for (int i = 0; i < 2; ++i)
    FPB_CHECK_ARG(o_strides[i] >= 0 && o_strides[i] < (int64_t(1) << 40), "out stride[%d]=%lld is out of range", i,
                  (long long)o_strides[i]);
  FPB_CHECK_ARG((reinterpret_cast<uintptr_t>(lse) & 3) == 0, "lse must be an aligned float pointer or NULL");
  FPB_CHECK_ARG(std::isfinite(sm_scale), "sm_scale must be finite");
  const DecodeShape s = decode_shape(batch, hq, hk, cache_dtype, max_pages, page_size);
  if (s.cluster == 0) {
    FPB_CHECK_ARG(s.units < (int64_t(1) << 31),
                  "too many tokens for one call: batch * num_kv_heads * max_pages * page_size (narrow the page table)");
    FPB_CHECK_ARG(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
                  "workspace must be a 256-byte aligned device pointer");
    FPB_CHECK_ARG((int64_t)workspace_bytes >= decode_ws_total(s), "workspace too small: %zu bytes given, %lld needed",
                  workspace_bytes, (long long)decode_ws_total(s));
    auto* ws = static_cast<uint8_t*>(workspace);
    A.desc = reinterpret_cast<int4*>(ws);
    A.part = reinterpret_cast<float*>(ws + decode_ws_part(s));
    A.ml = reinterpret_cast<float2*>(ws + decode_ws_ml(s));
  }
  A.q = static_cast<const uint8_t*>(q);
  A.out = static_cast<uint8_t*>(out);
  A.lse = lse;
  A.q_b = 2 * q_strides[0];
  A.q_h = 2 * q_strides[1];
  A.o_b = 2 * o_strides[0];
  A.o_h = 2 * o_strides[1];
  A.page_table = page_table;
  A.table_stride = table_stride;
  A.seq_lens = seq_lens;
  A.max_pages = max_pages;
  A.batch = batch;
  A.hq = hq;
  A.hk = hk;
  A.G = s.G;
  A.ngroups = s.ngroups;
  A.nh = s.nh;
  A.by_item = s.by_item;
  A.join_heads = s.join_heads;
  A.c = (float)(sm_scale * 1.4426950408889634);
  A.page16 = page_size % 16 == 0;
  auto st = static_cast<cudaStream_t>(stream);
  const bool bf16 = dtype == FPB_BF16, e4m3 = cache_dtype == FPB_E4M3, wide = s.nh > 8;
  if (bf16) {
    if (e4m3) return wide ? launch_decode<__nv_bfloat16, true, 2>(A, s, st) : launch_decode<__nv_bfloat16, true, 1>(A, s, st);
    return wide ? launch_decode<__nv_bfloat16, false, 2>(A, s, st) : launch_decode<__nv_bfloat16, false, 1>(A, s, st);
  }
  if (e4m3) return wide ? launch_decode<__half, true, 2>(A, s, st) : launch_decode<__half, true, 1>(A, s, st);
  return wide ? launch_decode<__half, false, 2>(A, s, st) : launch_decode<__half, false, 1>(A, s, st);
}

int fpb_paged_read_device_error(uint32_t* flags, void* stream) {
  FPB_CHECK_ARG(flags != nullptr, "flags is NULL");
  auto st = static_cast<cudaStream_t>(stream);
  static std::mutex one_at_a_time;  // g_paged_taken holds one reader's bits
  const std::lock_guard<std::mutex> lock(one_at_a_time);
  uint32_t h = 0;
  paged_take_err_kernel<<<1, 1, 0, st>>>();
  FPB_CUDA(cudaGetLastError());
  FPB_CUDA(cudaMemcpyFromSymbolAsync(&h, g_paged_taken, sizeof(h), 0, cudaMemcpyDeviceToHost, st));
  FPB_CUDA(cudaStreamSynchronize(st));
  *flags = h;
  return h == 0 ? FPB_OK : fail(FPB_EDEVICE, "device error bits 0x%x", h);
}

}  // extern "C"
