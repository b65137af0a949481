// Attention of one new token for each sequence over its pages of the cache (fp_paged.cu), split over the cache's length
// and joined.
//
//   s_j = sm_scale * q . k_j,   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   lse = m + log sum_j exp(s_j - m)
//
// for every sequence b and query head, j over the sequence's seq_lens[b] cached tokens; the G = hq / hk query heads of a
// KV head share its rows.  Each cached byte is read once (once for each group of at most 16 heads, where a KV head has more) and
// meets G flops (2-byte cache) or 2 G (e4m3), so the operator is bound by HBM; the arithmetic only has to stay out of the way.
//
// An item is (sequence, KV head, group of query heads: all G up to 16, equal groups of at most 16 above that); its tokens are
// cut into units of TT tokens for each warp of a CTA.  Lengths are read on the device (no host copy; a captured graph serves
// any lengths).
//
// Long sequences (paged_decode_kernel).  All items' units form one line, with one empty unit at the head of each item for
// what starting an item costs, and each of the CTAs that the GPU holds takes an equal piece of it, so ragged batches and
// single long sequences load the GPU alike.  A piece that covers a whole item writes its output; an item cut between pieces
// leaves unnormalised sums and their maxima in the workspace; a second kernel joins them in the order of the tokens.
// Short sequences (paged_decode_short_kernel): one cluster of 1 to 8 CTAs for each item, units dealt out in turn, joined
// through distributed shared memory.  No prefix sums, no workspace, no second kernel.
// Both join in an order that follows from the call's shapes (the table's width among them) and the lengths, with no atomics: the
// same call gives the same bits.
//
// A warp works alone on its own tiles of TT tokens (16 of a 16-bit cache, 32 of e4m3: 4 KB of K and of V each way) through
// a ring of kDecStages tiles filled by 16-byte cp.async, so loads are in flight all the time without block-wide barriers;
// warps meet once an item.  Where page_size is a multiple of 16, 16 tokens share a page and one table entry, fetched a tile
// ahead, gives their addresses; other page sizes look each row up.  Rows behind the end, or on a page that is not in the
// cache, are filled with zeros and their scores set to -inf: stale values there never reach the sums.
//
// Tensor cores.  S^T = K Q^T with the tokens as the 16 rows and 8 heads as the columns of mma.m16n8k16; out^T = V^T P^T
// with the channels as rows.  The small side of both products is the 8-wide one, so G <= 8 heads cost one pass where
// tcgen05's least tile would be mostly padding, and the operands need no staging beyond the ring.
//   * Scores, maxima, sums and outputs stay in fp32 registers.  The running maximum is reduced over the warp, and sums are
//     rescaled, only in tiles where some score exceeds it.
//   * P is split into two 16-bit parts (the value and its remainder) and multiplied twice: one part alone would leave errors
//     as large as the output's own rounding.  Only for an e4m3 cache with bf16 output is one part enough: fp16 products, an
//     eighth of the output's rounding (two parts there, of which the products' power slows the clock: 2 x 256K 92 us, 86 with
//     one; 33 x 16K 59.4 and 56.5; the output's distance from the 64-bit result 1% less).
//     Where V may hold infinities (16-bit caches) the first part is rounded towards zero and the second kept above zero, so
//     that both products of a weight and an infinity have its sign, as the weight's own has: a remainder of 0 or below 0 would
//     make a NaN of it.
//   * fp16 products: P is scaled by 2^15 (as the row sum is, so it cancels), which keeps weights down to 2^-29 of the
//     largest in fp16's normal range.
//   * e4m3: codes widen to fp16 exactly; q is scaled by a power of two to fill fp16's range; the token's K scale multiplies its
//     score and its V scale its weight.  These products must fit fp16, so the running maximum is that of score + log2(V scale)
//     and they reach 2^15; the sum of the weights goes by the same reference and is brought to [1, 2) when an item ends.
//     With weights relative to the largest score and V scales to the largest of any token, a row of small values behind one of
//     large values lost bits, and all of them from 2^39 on, even where the softmax gave the large ones no weight.  Scores
//     beyond 4096 need another reference (weigh_large); a warp that meets one begins its item again.
//
// Measured (calls in a row; of the measured 6.54 TB/s): 64 x up to 8192 tokens of 32/8 heads, bf16, 1.11 GB, 165 to 170 us (100%
// and more: reads alone pass a copy's rate); 1 x 131072, 0.54 GB, 84 us (98%); 2 x up to 262144 of 28/4 heads, e4m3, 0.53 GB,
// 86 to 88 us (92 to 94%; 82 at the clocks of a short run), 52% of the issue slots; 33 x up to 16001 of 28/4 heads, e4m3, 0.31
// GB, 56.8 us (82%; 53 at the clocks of a short run): 3 us from the launch to the first full stream (lengths, table, rows: three
// loads in turn), 3 us between the first CTA that ends and the last, 4 us for the join.  1 x 500 of 32/8 heads, 2 MB, 4.5 us: the
// launch 0.9, the same loads in turn and the warps' sums 1.8, the cluster's barrier and sums 1.8.
#include <cfloat>
#include <type_traits>

#include "fp_common.cuh"

namespace fpb {

constexpr int kDecStages = 2;
constexpr int kDecTileBytes = 4096;  // one warp's tile of K or of V
constexpr int kDecScaleBytes = 128;  // e4m3: scales of a tile's 32 rows of K or of V
constexpr int kDecStageBytes = 2 * (kDecTileBytes + kDecScaleBytes);
constexpr int kDecRingBytes = kDecStages * kDecStageBytes;
// CTAs of narrow (4 warps) and wide form (as many as the registers hold: one CTA an SM), by 8s of heads of an item.
constexpr int kNarrow = 4;
constexpr int wide_warps(int nt) { return nt == 1 ? 12 : 8; }
constexpr int dec_ctas_per_sm(int nt, int warps) { return wide_warps(nt) / warps; }
constexpr int dec_smem_bytes(int warps) { return warps * kDecRingBytes; }
constexpr int kDecMaxCluster = 8;  // clusters are powers of two: each divides the 8 NT heads of an item
constexpr int kJoinThreads = 256;
constexpr float kLn2 = 0.6931471805599453f;

struct DecodeArgs {
  PagedCache C;
  const uint8_t* q;
  uint8_t* out;
  float* lse;                        // may be null; contiguous (batch, hq)
  int64_t q_b, q_h, o_b, o_h;        // bytes
  const int* page_table;
  int64_t table_stride;
  const int* seq_lens;
  int page16;                        // page_size is a multiple of 16
  int max_pages, batch, hq, hk;
  int G, ngroups, nh;                // query heads of a KV head, groups of them, heads of a group (the last may have fewer)
  float c;                           // sm_scale * log2(e)
  int by_item;                       // desc is indexed by item (else by the piece that begins the item)
  int join_heads;                    // heads of a CTA of the second kernel
  int4* desc;                        // {b, KV head * groups + group, first piece, pieces (0: nothing to join)}
  float* part;                       // [2 * piece + slot][nh][128]; slot 1 where the piece begins the item, else 0
  float2* ml;                        // [2 * piece + slot][nh] {maximum (log2 units), sum}
};

// 16 bytes of the cache (`bytes` of them, then zeros) to shared memory.  Cached rows pass through L2 once: evicted first, they
// leave it to the tables, lengths and partial sums (28/4 heads, 33 x up to 16001 tokens of e4m3: 57 us without, 53 with).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes),
               "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float lds(uint32_t addr) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// D += A B with A 16x16, B 16x8 (T = bf16 or fp16), fp32 accumulators
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (DT<T>::is_bf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// First of a cluster's two barriers: every CTA has started, so its shared memory may be written from the others.
__device__ __forceinline__ void cluster_started_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_started_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// Second: what the CTAs wrote into one another is there.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Writes the float at this CTA's shared address `addr` in CTA `rank` of the cluster.
__device__ __forceinline__ void st_cluster(uint32_t addr, int rank, float v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}

// A pair of weights as two 16-bit parts whose sum they are, to 2^-16 (bf16: truncated, and a remainder of 2^-23 at the least) or
// 2^-21 and 2^-39 of the largest weight (fp16, which holds weights times 2^15: rounded towards zero, and a remainder of one step
// at the least).  A weight that is not zero has two parts above zero (fp16: one of 2^-39 or more).
template <typename T>
__device__ __forceinline__ void split_weights(float x, float y, uint32_t& first, uint32_t& rest) {
  if constexpr (DT<T>::is_bf16) {
    constexpr float kBelowOne = 1.f - 1.1920928955078125e-07f;
    first = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    rest = DT<T>::pack(fmaf(DT<T>::lo(first), -kBelowOne, x), fmaf(DT<T>::hi(first), -kBelowOne, y));
  } else {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(first) : "f"(y), "f"(x));
    const uint32_t r = DT<T>::pack(x - DT<T>::lo(first), y - DT<T>::hi(first));
    asm("max.f16x2 %0, %1, %2;" : "=r"(rest) : "r"(r), "r"(0x00010001u));
  }
}

__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// Tokens of sequence b; a length outside [0, room] is reported and counts as 0.
__device__ __forceinline__ int seq_len_of(const DecodeArgs& A, int b) {
  const int len = A.seq_lens[b];
  if (len < 0 || len > (int64_t)A.max_pages * A.C.page_size) {
    raise_error(&g_paged_err, kErrBadLength);
    return 0;
  }
  return len;
}

// T: type of q and out; kE4m3: codes in the cache (else T); NT: groups of 8 heads of an item.
template <typename T, bool kE4m3, int NT>
struct DecodeWarp {
  using MT = typename std::conditional<kE4m3, __half, T>::type;  // type of the products
  static constexpr int TT = kE4m3 ? 32 : 16;                     // tokens of a tile
  static constexpr int MTILES = TT / 16;
  static constexpr int kRowBytes = kDecTileBytes / TT;
  static constexpr int kChunks = kRowBytes / 16;  // 16-byte pieces of a row
  static constexpr uint32_t kFull = TT == 32 ? 0xFFFFFFFFu : 0xFFFFu;
  static constexpr bool kSplitP = !(kE4m3 && DT<T>::is_bf16);    // P as two parts
  static constexpr float kShift = DT<MT>::is_bf16 ? 0.f : 15.f;  // log2 of the factor of P and l
  static constexpr float kLarge = 4096.f;                        // e4m3: scores beyond are weighed by weigh_large
  // V scales as the running maximum takes them: P is kept finite beyond, and the sum of 2^31 weights below.
  static constexpr float kLeastScale = 8.271806125530277e-25f;   // 2^-80
  static constexpr float kLargestScale = 1.329227995784916e36f;  // 2^120

  uint32_t ring;  // shared address of this warp's ring
  int lane;
  uint32_t qf[NT][8][2];      // q as the B operand
  float qc[NT][2];            // factor of this thread's two columns (heads 2t, 2t + 1)
  float o[NT][8][4];          // out^T: 16 channels x 8 heads a tile
  float m[NT][2], l[NT][2];   // running maximum (e4m3: of score + log2 of V's scale) and this thread's share of the sum

  // q's rows as they are in memory.  An e4m3 row gives a thread elements 4t .. 4t+3 of each 16: they take the places 2t,
  // 2t+1, 2t+8, 2t+9 of the product's inner dimension, in q as in K.
  __device__ __forceinline__ void load_q(const DecodeArgs& A, const uint8_t* q, int heads) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool ok = n * 8 + g < heads;
      const uint8_t* row = q + (n * 8 + g) * A.q_h;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if constexpr (!kE4m3) {
          qf[n][k][0] = ok ? *reinterpret_cast<const uint32_t*>(row + 32 * k + 4 * t) : 0u;
          qf[n][k][1] = ok ? *reinterpret_cast<const uint32_t*>(row + 32 * k + 4 * t + 16) : 0u;
        } else {
          const uint2 x = ok ? *reinterpret_cast<const uint2*>(row + 32 * k + 8 * t) : make_uint2(0u, 0u);
          qf[n][k][0] = x.x;
          qf[n][k][1] = x.y;
        }
      }
    }
  }
  // q in the products' type and the factors of the scores.
  __device__ __forceinline__ void convert_q(const DecodeArgs& A) {
    const int t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f = 1.f;
      if constexpr (kE4m3 && DT<T>::is_bf16) {
        uint32_t mx = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) mx = absmax2(absmax2(mx, qf[n][k][0]), qf[n][k][1]);
        mx = max(mx & 0xFFFFu, mx >> 16);
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // power of two that brings the row's largest magnitude to [2^14, 2^15), which leaves elements 2^28 times smaller in
        // fp16's normal range; inf and NaN pass as they are
        const int e = max(-120, (int)(mx >> 7) - 127 - 14);
        const float down = exp2i(-e);
        f = exp2i(e);
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            qf[n][k][j] = DT<__half>::pack(DT<T>::lo(qf[n][k][j]) * down, DT<T>::hi(qf[n][k][j]) * down);
      }
      qc[n][0] = A.c * __shfl_sync(0xffffffffu, f, 8 * t);
      qc[n][1] = A.c * __shfl_sync(0xffffffffu, f, 8 * t + 4);
    }
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
    }
  }

  // Table entries of the tile at `tok` (one for each 16 tokens).  Entries behind the sequence may be read, never used.
  __device__ __forceinline__ void load_pages(const DecodeArgs& A, const int* table, int tok, int (&page)[MTILES]) {
#pragma unroll
    for (int j = 0; j < MTILES; ++j) {
      const int p = A.C.page_of(tok + 16 * j);
      page[j] = p < A.max_pages ? table[p] : -1;
    }
  }

  // Starts the copies of tokens [tok, tok + TT) below `end` into ring slot `stage`.  valid: bit r set where row r is there.
  // The scales go to shared memory with the rows: loaded into registers a tile ahead, they were waited for together with
  // the loads of the tile behind them (4 x 8100 tokens of 32/8 heads, e4m3: 18.3 us so, 17.0 this way).
  __device__ __forceinline__ void issue(const DecodeArgs& A, const int* table, int h, int tok, int end,
                                        int stage, const int (&page)[MTILES], uint32_t& valid) {
    constexpr int kRowsPer = 32 / kChunks;  // rows of one copy instruction of the warp
    const uint32_t kd = ring + stage * kDecStageBytes, vd = kd + kDecTileBytes;
    const uint32_t sd = kd + 2 * kDecTileBytes + 4 * lane;
    const int ch = lane % kChunks, r0 = lane / kChunks;
    if (A.page16) {
      valid = 0;
#pragma unroll
      for (int j = 0; j < MTILES; ++j) {
        const int t0 = tok + 16 * j;
        int rows = max(0, min(16, end - t0));
        unsigned pg = page[j];
        if (rows > 0 && pg >= (unsigned)A.C.num_pages) {
          raise_error(&g_paged_err, kErrBadPage);
          rows = 0;
        }
        if (rows == 0) pg = 0;
        const int at = rows == 0 ? 0 : t0 - A.C.page_of(t0) * A.C.page_size;
        valid |= ((1u << rows) - 1u) << (16 * j);
        const uint64_t off = A.C.rows.at(pg, at + r0, h) * 16 + ch * 16;
        const uint8_t* kp = A.C.k + off;
        const uint8_t* vp = A.C.v + off;
        const uint64_t step = (uint64_t)A.C.rows.tok * (16 * kRowsPer);
#pragma unroll
        for (int i = 0; i < 16 / kRowsPer; ++i) {
          const int r = i * kRowsPer + r0, row = 16 * j + r;
          const uint32_t d = row * kRowBytes + ((ch ^ (row & 7)) << 4);
          const int bytes = r < rows ? 16 : 0;  // rows behind the end lie on the same page
          cp_async16(kd + d, kp, bytes);
          cp_async16(vd + d, vp, bytes);
          kp += step;
          vp += step;
        }
        if constexpr (kE4m3) {
          if (lane / 16 == j) {
            const uint64_t so = A.C.scales.at(pg, at + lane % 16, h);
            const int bytes = lane % 16 < rows ? 4 : 0;
            cp_async4(sd, A.C.k_scale + so, bytes);
            cp_async4(sd + kDecScaleBytes, A.C.v_scale + so, bytes);
          }
        }
      }
      return;
    }
    const int my = tok + lane % TT;
    int64_t off = -1;
    uint64_t so = 0;
    if (my < end) {
      const int p = A.C.page_of(my), at = my - p * A.C.page_size, pg = table[p];
      if ((unsigned)pg < (unsigned)A.C.num_pages) {
        off = (int64_t)(A.C.rows.at(pg, at, h) * 16);
        if constexpr (kE4m3) so = A.C.scales.at(pg, at, h);
      } else {
        raise_error(&g_paged_err, kErrBadPage);
      }
    }
    if constexpr (kE4m3) {
      cp_async4(sd, A.C.k_scale + so, off < 0 ? 0 : 4);
      cp_async4(sd + kDecScaleBytes, A.C.v_scale + so, off < 0 ? 0 : 4);
    }
    valid = __ballot_sync(0xffffffffu, off >= 0);
    if constexpr (TT == 16) valid &= 0xFFFFu;
#pragma unroll 1
    for (int i = 0; i < TT / kRowsPer; ++i) {
      const int r = i * kRowsPer + r0;
      const int64_t ro = __shfl_sync(0xffffffffu, off, r);
      const uint32_t d = r * kRowBytes + ((ch ^ (r & 7)) << 4);
      const int64_t src = ro < 0 ? 0 : ro + ch * 16;
      cp_async16(kd + d, A.C.k + src, ro < 0 ? 0 : 16);
      cp_async16(vd + d, A.C.v + src, ro < 0 ? 0 : 16);
    }
  }

  // Scales of the row of a tile that this thread's elements (i, h) of s belong to: g + 8 h + 16 i.
  __device__ __forceinline__ float k_scale(int stage, int i, int h) const {
    return lds(ring + stage * kDecStageBytes + 2 * kDecTileBytes + 4 * (16 * i + 8 * h + (lane >> 2)));
  }
  __device__ __forceinline__ float v_scale(int stage, int i, int h) const {
    return lds(ring + stage * kDecStageBytes + 2 * kDecTileBytes + kDecScaleBytes + 4 * (16 * i + 8 * h + (lane >> 2)));
  }
  __device__ __forceinline__ float log_v_scale(int stage, int i, int h) const {
    return __log2f(fminf(fmaxf(fabsf(v_scale(stage, i, h)), kLeastScale), kLargestScale));
  }
  // Whether that row is there.
  __device__ __forceinline__ bool there(uint32_t valid, int i, int h) const { return (valid >> (16 * i + 8 * h + (lane >> 2))) & 1u; }
  // The largest of a column's rows.
  static __device__ __forceinline__ float max_rows(float x) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
  }
  __device__ __forceinline__ void rescale(int n, float (&f)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) l[n][j] *= f[j];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[n][i][j] *= f[j & 1];
  }

  // Products of a tile's keys and q, times the factor of q: scores in log2 units, of an e4m3 row without its K scale.
  __device__ __forceinline__ void scores(int stage, float (&s)[NT][MTILES][4]) {
    const uint32_t kd = ring + stage * kDecStageBytes;
    {
      float s2[NT][4];  // second chain of products of a 16-token tile (32 tokens have two as it is)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s2[n][j] = 0.f;
#pragma unroll
          for (int i = 0; i < MTILES; ++i) s[n][i][j] = 0.f;
        }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t a[4];
        if constexpr (!kE4m3) {
          const int r = lane & 15, ch = 2 * k + (lane >> 4);
          ldsm4(a, kd + r * kRowBytes + ((ch ^ (r & 7)) << 4));
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma16816<MT>(k & 1 ? s2[n] : s[n][0], a[0], a[1], a[2], a[3], qf[n][k][0], qf[n][k][1]);
        } else {
          ldsm4(a, kd + lane * kRowBytes + ((k ^ (lane & 7)) << 4));
#pragma unroll
          for (int i = 0; i < MTILES; ++i) {
            const uint32_t a0 = e4m3x2_to_f16x2(a[2 * i]), a2 = e4m3x2_to_f16x2(a[2 * i] >> 16);
            const uint32_t a1 = e4m3x2_to_f16x2(a[2 * i + 1]), a3 = e4m3x2_to_f16x2(a[2 * i + 1] >> 16);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<MT>(s[n][i], a0, a1, a2, a3, qf[n][k][0], qf[n][k][1]);
          }
        }
      }
      if constexpr (!kE4m3) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][0][j] += s2[n][j];
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][i][j] *= qc[n][j & 1];
  }

  // Scores of a tile to weights.  e4m3: false, with nothing done, where the running maximum would leave [-kLarge, kLarge].
  __device__ __forceinline__ bool weigh(int stage, uint32_t valid, float (&s)[NT][MTILES][4]) {
    if constexpr (kE4m3) {
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float kf = k_scale(stage, i, h);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) s[n][i][2 * h + j] *= kf;
        }
    }
    if (valid != kFull) {
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (!there(valid, i, h)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) s[n][i][2 * h] = s[n][i][2 * h + 1] = -INFINITY;
          }
    }
    // the largest of this thread's rows g, g + 8 (+ 16 i) for its columns 2t + j
    float mx[NT][2];
#pragma unroll
    for (int i = 0; i < MTILES; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float lv = kE4m3 ? log_v_scale(stage, i, h) : 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float x = kE4m3 ? s[n][i][2 * h + j] + lv : s[n][i][2 * h + j];
            mx[n][j] = i + h == 0 ? x : fmaxf(mx[n][j], x);
          }
      }
    bool moved = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) moved |= mx[n][0] > m[n][0] || mx[n][1] > m[n][1];
    if (__any_sync(0xffffffffu, moved)) {
      bool large = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mx[n][j] = max_rows(mx[n][j]);
          // e4m3: on a grid of 2^-6, so that neither 15 nor the sum's exponent changes its low bits on the way to the lse
          if constexpr (kE4m3) mx[n][j] = ceilf(mx[n][j] * 64.f) * (1.f / 64.f);
          mx[n][j] = fmaxf(m[n][j], mx[n][j]);
          large |= fabsf(finite_or_zero(mx[n][j])) > kLarge;
        }
      if (kE4m3 && __any_sync(0xffffffffu, large)) return false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          f[j] = ex2_approx(m[n][j] - finite_or_zero(mx[n][j]));
          m[n][j] = mx[n][j];
        }
        rescale(n, f);
      }
    }
#pragma unroll
    for (int i = 0; i < MTILES; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float& x = s[n][i][2 * h + j];
            x = ex2_approx(kE4m3 ? x - (finite_or_zero(m[n][j]) - kShift) : (x - finite_or_zero(m[n][j])) + kShift);
            l[n][j] += x;
          }
    return true;
  }

  // The same for e4m3 scores of any size.  Above some millions what is added to a score is rounded away, so the reference has two
  // parts, m + w: m the largest score, w the log2 that the largest product of a weight and a V scale has above it, less kShift.
  // Scores are taken off m with one rounding.  (In every tile this would cost 33 x 16K 2 us of 53.)
  __device__ __forceinline__ void weigh_large(int stage, uint32_t valid, float (&s)[NT][MTILES][4], float (&w)[NT][2]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = m[n][j], y = -INFINITY;
#pragma unroll
        for (int i = 0; i < MTILES; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (there(valid, i, h)) x = fmaxf(x, s[n][i][2 * h + j] * k_scale(stage, i, h));
        x = max_rows(x);
        const float up = x - m[n][j];
#pragma unroll
        for (int i = 0; i < MTILES; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& d = s[n][i][2 * h + j];
            d = there(valid, i, h) ? fmaf(d, k_scale(stage, i, h), -x) : -INFINITY;
            y = fmaxf(y, d + log_v_scale(stage, i, h));
          }
        const float wn = fmaxf(w[n][j] - up, max_rows(y) - kShift);
        f[j] = ex2_approx(w[n][j] - up - wn);
        m[n][j] = x;
        w[n][j] = wn;
#pragma unroll
        for (int i = 0; i < MTILES; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) s[n][i][2 * h + j] = ex2_approx(s[n][i][2 * h + j] - wn);
      }
      rescale(n, f);
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) l[n][j & 1] += s[n][i][j];
    }
  }

  // Weights times the tile's values.
  __device__ __forceinline__ void products(int stage, const float (&s)[NT][MTILES][4]) {
    const uint32_t vd = ring + stage * kDecStageBytes + kDecTileBytes;
    uint32_t pb[NT][MTILES][2], pl[NT][MTILES][2];
#pragma unroll
    for (int i = 0; i < MTILES; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float vs = kE4m3 ? v_scale(stage, i, h) : 1.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float p[2] = {s[n][i][2 * h] * vs, s[n][i][2 * h + 1] * vs};
          uint32_t hi, lo;
          if constexpr (!kE4m3) {
            split_weights<MT>(p[0], p[1], hi, lo);
          } else {
            hi = DT<MT>::pack(p[0], p[1]);
            if constexpr (kSplitP) lo = DT<MT>::pack(p[0] - DT<MT>::lo(hi), p[1] - DT<MT>::hi(hi));
          }
          pb[n][i][h] = transpose8x8(hi);
          if constexpr (kSplitP) pl[n][i][h] = transpose8x8(lo);
        }
      }
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // 16 channels
      uint32_t a[4];
      if constexpr (!kE4m3) {
        const int r = (lane & 7) + ((lane >> 4) << 3), ch = 2 * i + ((lane >> 3) & 1);
        ldsm4_trans(a, vd + r * kRowBytes + ((ch ^ (r & 7)) << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816<MT>(o[n][i], a[0], a[1], a[2], a[3], pb[n][0][0], pb[n][0][1]);
          if constexpr (kSplitP) mma16816<MT>(o[n][i], a[0], a[1], a[2], a[3], pl[n][0][0], pl[n][0][1]);
        }
      } else {
        // transposed pairs of codes: {token 2t: channels 2g, 2g+1; token 2t+1: channels 2g, 2g+1}; channel 2g becomes
        // row g of the product and channel 2g+1 row g + 8
        ldsm4_trans(a, vd + lane * kRowBytes + ((i ^ (lane & 7)) << 4));
#pragma unroll
        for (int k = 0; k < MTILES; ++k) {
          const uint32_t x = __byte_perm(a[2 * k], 0, 0x3120), y = __byte_perm(a[2 * k + 1], 0, 0x3120);
          const uint32_t a0 = e4m3x2_to_f16x2(x), a1 = e4m3x2_to_f16x2(x >> 16);
          const uint32_t a2 = e4m3x2_to_f16x2(y), a3 = e4m3x2_to_f16x2(y >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816<MT>(o[n][i], a0, a1, a2, a3, pb[n][k][0], pb[n][k][1]);
            if constexpr (kSplitP) mma16816<MT>(o[n][i], a0, a1, a2, a3, pl[n][k][0], pl[n][k][1]);
          }
        }
      }
    }
  }

  // False where weigh refused: the item's scores are large.
  __device__ __forceinline__ bool consume(int stage, uint32_t valid) {
    float s[NT][MTILES][4];
    scores(stage, s);
    if (!weigh(stage, valid, s)) return false;
    products(stage, s);
    return true;
  }

  // All of this warp's tiles of an item: tokens [tok + i * step, + TT) below min(end, the sequence's length).  The first
  // table entries and q are on their way before the length is needed.  kAhead: the next tile is asked for before, not after,
  // the wait for this one.  That shortens a warp's chain of tiles (256 x up to 600 tokens 19.6 -> 18.3 us, 1 x 8192 11.8 ->
  // 10.6) but puts more in flight than long streams bear (64 x up to 8192, bf16: 168 -> 174 us).
  template <bool kAhead>
  __device__ __forceinline__ void run(const DecodeArgs& A, int b, int h, int head0, int heads, int tok, int step, int end) {
    const int* table = A.page_table + b * A.table_stride;
    int page[MTILES];
    load_pages(A, table, tok, page);
    load_q(A, A.q + b * A.q_b + head0 * A.q_h, heads);
    const int n = end > tok ? (end - tok + step - 1) / step : 0;
    uint32_t valid[kDecStages];
#pragma unroll
    for (int i = 0; i < kDecStages - 1; ++i) {
      if (i < n) {
        int cur[MTILES];
#pragma unroll
        for (int j = 0; j < MTILES; ++j) cur[j] = page[j];
        if (i + 1 < n) load_pages(A, table, tok + (i + 1) * step, page);
        issue(A, table, h, tok + i * step, end, i, cur, valid[i]);
      }
      cp_async_commit();
    }
    convert_q(A);
    reset();
    for (int i0 = 0; i0 < n; i0 += kDecStages) {
#pragma unroll
      for (int j = 0; j < kDecStages; ++j) {
        if (i0 + j < n) {
          if constexpr (!kAhead) {
            cp_async_wait<kDecStages - 2>();
            __syncwarp();
          }
          constexpr int kNext = kDecStages - 1;
          const int st = (j + kNext) % kDecStages, nx = i0 + j + kNext;
          if (nx < n) {
            int cur[MTILES];
#pragma unroll
            for (int x = 0; x < MTILES; ++x) cur[x] = page[x];
            if (nx + 1 < n) load_pages(A, table, tok + (nx + 1) * step, page);
            issue(A, table, h, tok + nx * step, end, st, cur, valid[st]);
          }
          cp_async_commit();
          if constexpr (kAhead) {
            cp_async_wait<kDecStages - 1>();
            __syncwarp();
          }
          if (!consume(j, valid[j])) goto large;
          __syncwarp();
        }
      }
    }
    cp_async_wait<0>();
    __syncwarp();
    return;
  large:
    if constexpr (kE4m3) {  // once more from the first tile, one after another
      cp_async_wait<0>();
      __syncwarp();
      reset();
      float w[NT][2];
#pragma unroll
      for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) m[k][j] = w[k][j] = -FLT_MAX;
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        load_pages(A, table, tok + i * step, page);
        issue(A, table, h, tok + i * step, end, 0, page, valid[0]);
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
        float s[NT][MTILES][4];
        scores(0, s);
        weigh_large(0, valid[0], s, w);
        products(0, s);
        __syncwarp();
      }
      // sums relative to m, as scores are: what is added to m now would be rounded away
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        float f[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bool none = w[k][j] == -FLT_MAX;
          f[j] = none ? 1.f : ex2_approx(w[k][j] + kShift);
          if (none) m[k][j] = -INFINITY;
        }
        rescale(k, f);
      }
    }
  }

  // Sums and maxima into shared memory: rows of 132 floats for each head (conflict-free), {maximum, sum} beside them.
  __device__ __forceinline__ void store(float* so, float2* sml) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = l[n][j];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        const int h = n * 8 + 2 * t + j;
        // relative to m: the factor 2^kShift comes off the sums, not m.  e4m3 sums of scores that are not large are first brought
        // to [1, 2), as they may be far from it.
        float f = exp2i(-(int)kShift), top = m[n][j];
        if (kE4m3 && fabsf(top) <= kLarge) {
          const int e = max(-120, min((int)(__float_as_uint(x) >> 23) - 127, 120));
          f = exp2i(-e);
          top += (float)e - kShift;
        }
        if (g == 0) sml[h] = make_float2(top, x * f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d0 = 16 * i + (kE4m3 ? 2 * g : g), d1 = 16 * i + (kE4m3 ? 2 * g + 1 : g + 8);
          so[h * 132 + d0] = o[n][i][j] * f;
          so[h * 132 + d1] = o[n][i][2 + j] * f;
        }
      }
  }
};

// Joins the warps' sums of head i at channel d: {sum of weights times v, sum of weights, maximum}.
template <int kWarps, int NT>
__device__ __forceinline__ void merge_warps(const uint8_t* smem, const float2 (&s_ml)[kWarps][8 * NT], int i, int d, float& x,
                                            float& l, float& mx) {
  mx = -INFINITY;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) mx = fmaxf(mx, s_ml[k][i].x);
  const float ref = finite_or_zero(mx);
  l = x = 0.f;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) {
    const float f = ex2_approx(s_ml[k][i].x - ref);
    l += f * s_ml[k][i].y;
    x += f * reinterpret_cast<const float*>(smem + k * kDecRingBytes)[i * 132 + d];
  }
}

template <typename T>
__device__ __forceinline__ void write_head(const DecodeArgs& A, int b, int head, int d, float x, float l, float mx) {
  reinterpret_cast<T*>(A.out + b * A.o_b + head * A.o_h)[d] = DT<T>::from_f(l == 0.f ? 0.f : x / l);
  if (A.lse && d == 0) A.lse[(int64_t)b * A.hq + head] = l == 0.f ? -INFINITY : (mx + log2f(l)) * kLn2;
}

// Equal cuts of `total` units into `n` pieces: piece i starts at i * q + min(i, r).
struct Cut {
  int q, r;
  __device__ __forceinline__ Cut(int total, int n) : q(total / n), r(total - q * n) {}
  __device__ __forceinline__ int start(int i) const { return i * q + min(i, r); }
  __device__ __forceinline__ int piece(int t) const { return t < r * (q + 1) ? t / (q + 1) : r + (t - r * (q + 1)) / q; }
};

template <typename T, bool kE4m3, int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, dec_ctas_per_sm(NT, kWarps)) paged_decode_kernel(const DecodeArgs A) {
  using W = DecodeWarp<T, kE4m3, NT>;
  constexpr int kUnit = kWarps * W::TT;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 s_ml[kWarps][8 * NT];
  static_assert(8 * NT * 132 * 4 <= kDecRingBytes, "a warp's sums fit its ring");

  await_stream();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, d = tid % kHeadDim;
  const int HH = A.hk * A.ngroups, v = blockIdx.x;

  // ---- this CTA's piece, found by every warp for itself: prefix sums of the sequences' units.  The host has checked that
  // all units together stay below 2^31.
  auto units_of = [](int len) { return 1 + (len + kUnit - 1) / kUnit; };
  const int per = (A.batch + 31) / 32;
  const int b_lo = min(lane * per, A.batch), b_hi = min(b_lo + per, A.batch);
  int mine = 0;
#pragma unroll 8
  for (int i = b_lo; i < b_hi; ++i) mine += units_of(seq_len_of(A, i));
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += x;
  }
  const int total = __shfl_sync(0xffffffffu, incl, 31) * HH;
  const int pieces = min((int)gridDim.x, total);
  if (!A.by_item && tid == 0) A.desc[v] = make_int4(0, 0, 0, 0);
  if (v >= pieces) return;
  const Cut cut(total, pieces);
  int t = cut.start(v);
  const int t_end = cut.start(v + 1);
  int b = b_lo, len = 0, base = (incl - mine) * HH;
  const bool here = base <= t && t < incl * HH;  // one lane
  if (here) {
    while (true) {
      len = seq_len_of(A, b);
      const int n = units_of(len) * HH;
      if (t < base + n) break;
      base += n;
      ++b;
    }
  }
  const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  b = __shfl_sync(0xffffffffu, b, src);
  len = __shfl_sync(0xffffffffu, len, src);
  base = __shfl_sync(0xffffffffu, base, src);
  int units = units_of(len);
  int hh = (t - base) / units;
  int u = (t - base) - hh * units;

  W w;
  w.lane = lane;
  w.ring = smem_u32(smem) + warp * kDecRingBytes;
  float* const so = reinterpret_cast<float*>(smem + warp * kDecRingBytes);

  while (t < t_end) {
    const int u_end = min(units, u + (t_end - t));
    const int h = hh / A.ngroups, grp = hh - h * A.ngroups;
    const int head0 = h * A.G + grp * A.nh, heads = min(A.nh, A.G - grp * A.nh);
    // units u .. u_end hold the tokens [(u - 1) kUnit, (u_end - 1) kUnit); the first of an item none
    w.template run<false>(A, b, h, head0, heads, max(u - 1, 0) * kUnit + warp * W::TT, kUnit,
          min(len, (u_end - 1) * kUnit));
    w.store(so, s_ml[warp]);
    __syncthreads();

    const bool whole = u == 0 && u_end == units;
    const int64_t slot = 2 * v + (u == 0 ? 1 : 0);
    for (int i = tid / kHeadDim; i < heads; i += kWarps * 32 / kHeadDim) {
      float x, l, mx;
      merge_warps<kWarps, NT>(smem, s_ml, i, d, x, l, mx);
      if (whole) {
        write_head<T>(A, b, head0 + i, d, x, l, mx);
      } else {
        A.part[(slot * A.nh + i) * kHeadDim + d] = x;
        if (d == 0) A.ml[slot * A.nh + i] = make_float2(mx, l);
      }
    }
    if (u == 0 && tid == 0 && (A.by_item || !whole)) {
      const int v1 = cut.piece(t + units - 1);  // of the item's last unit
      A.desc[A.by_item ? b * HH + hh : v] = make_int4(b, hh, v, v1 > v ? v1 - v + 1 : 0);
    }
    __syncthreads();

    t += u_end - u;
    u = 0;
    if (++hh == HH) {
      hh = 0;
      if (++b < A.batch) {
        len = seq_len_of(A, b);
        units = units_of(len);
      }
    }
  }
}

// One item for each cluster of `cluster` CTAs (1, 2, 4 or 8); CTA r takes the units r, r + cluster, ...  Head i is joined by CTA
// i % cluster, into whose shared memory the others write their sums (written rather than fetched: one trip, and no CTA has to
// stay for its readers).
template <typename T, bool kE4m3, int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, dec_ctas_per_sm(NT, kWarps)) paged_decode_short_kernel(const DecodeArgs A, int cluster) {
  using W = DecodeWarp<T, kE4m3, NT>;
  constexpr int kUnit = kWarps * W::TT;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 s_ml[kWarps][8 * NT];
  // sums and {maximum, sum} from CTA k of the heads that this one joins: row k * own + j is head rank + j * cluster
  __shared__ float s_x[8 * NT][kHeadDim];
  __shared__ float2 s_cta[8 * NT];
  if (cluster > 1) cluster_started_arrive();
  await_stream();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, d = tid % kHeadDim;
  const int item = blockIdx.x / cluster, rank = blockIdx.x - item * cluster;
  const int HH = A.hk * A.ngroups, b = item / HH, hh = item - b * HH;
  const int h = hh / A.ngroups, grp = hh - h * A.ngroups;
  const int head0 = h * A.G + grp * A.nh, heads = min(A.nh, A.G - grp * A.nh);
  const int own = (heads + cluster - 1) / cluster;  // heads of a CTA; cluster divides 8 NT, so cluster * own <= 8 NT rows
  W w;
  w.lane = lane;
  w.ring = smem_u32(smem) + warp * kDecRingBytes;
  w.template run<true>(A, b, h, head0, heads, rank * kUnit + warp * W::TT, cluster * kUnit, seq_len_of(A, b));
  w.store(reinterpret_cast<float*>(smem + warp * kDecRingBytes), s_ml[warp]);
  __syncthreads();
  if (cluster > 1) cluster_started_wait();
  for (int i = tid / kHeadDim; i < heads; i += kWarps * 32 / kHeadDim) {
    float x, l, mx;
    merge_warps<kWarps, NT>(smem, s_ml, i, d, x, l, mx);
    if (cluster == 1) {
      write_head<T>(A, b, head0 + i, d, x, l, mx);
    } else {
      const int j = i / cluster, to = i - j * cluster, row = rank * own + j;
      st_cluster(smem_u32(&s_x[row][d]), to, x);
      if (d == 0) {
        st_cluster(smem_u32(&s_cta[row].x), to, mx);
        st_cluster(smem_u32(&s_cta[row].y), to, l);
      }
    }
  }
  if (cluster == 1) return;
  cluster_sync();
  for (int j = tid / kHeadDim; rank + j * cluster < heads; j += kWarps * 32 / kHeadDim) {
    float mx = -INFINITY;
    for (int k = 0; k < cluster; ++k) mx = fmaxf(mx, s_cta[k * own + j].x);
    const float ref = finite_or_zero(mx);
    float l = 0.f, x = 0.f;
    for (int k = 0; k < cluster; ++k) {
      const float2 ml = s_cta[k * own + j];
      const float f = ex2_approx(ml.x - ref);
      l += f * ml.y;
      x += f * s_x[k * own + j][d];
    }
    write_head<T>(A, b, head0 + rank + j * cluster, d, x, l, mx);
  }
}

__device__ __forceinline__ void scale4(float4& x, float f) { x = make_float4(x.x * f, x.y * f, x.z * f, x.w * f); }
__device__ __forceinline__ void add4(float4& x, float f, const float4& p) {
  x.x += f * p.x;
  x.y += f * p.y;
  x.z += f * p.z;
  x.w += f * p.w;
}

// Joins the pieces of the item of desc[blockIdx.x], heads [blockIdx.y * join_heads, + join_heads).  A warp takes one head and
// every parts-th piece, four of them and their maxima under way at a time; the parts meet in shared memory.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_decode_join_kernel(const DecodeArgs A) {
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ float s_x[kWarps][kHeadDim];
  __shared__ float2 s_ml[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int parts = kWarps / A.join_heads;  // join_heads <= kWarps
  const int part = warp / A.join_heads, i = blockIdx.y * A.join_heads + warp % A.join_heads;
  await_stream();
  const int4 d = A.desc[blockIdx.x];
  const int n = d.w;
  if (n == 0) return;
  const int b = d.x, h = d.y / A.ngroups, grp = d.y - h * A.ngroups;
  const int head0 = h * A.G + grp * A.nh, heads = min(A.nh, A.G - grp * A.nh);
  auto slot = [&](int k) { return (int64_t)(2 * (d.z + k) + (k == 0 ? 1 : 0)) * A.nh + i; };
  const bool mine = part < parts && i < heads;
  float mx = -INFINITY, l = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (mine) {
    constexpr int kBatch = 4;
    for (int k0 = part; k0 < n; k0 += kBatch * parts) {
      float2 ml[kBatch];
      float4 p[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int k = k0 + j * parts;
        ml[j] = k < n ? A.ml[slot(k)] : make_float2(-INFINITY, 0.f);
        p[j] = k < n ? reinterpret_cast<const float4*>(A.part + slot(k) * kHeadDim)[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float top = mx;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) top = fmaxf(top, ml[j].x);
      const float ref = finite_or_zero(top), f0 = ex2_approx(mx - ref);
      mx = top;
      l *= f0;
      scale4(x, f0);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float f = ex2_approx(ml[j].x - ref);
        l += f * ml[j].y;
        add4(x, f, p[j]);
      }
    }
    reinterpret_cast<float4*>(s_x[warp])[lane] = x;
    if (lane == 0) s_ml[warp] = make_float2(mx, l);
  }
  __syncthreads();
  if (!mine || part != 0) return;
  float top = mx;
  for (int k = 1; k < parts; ++k) top = fmaxf(top, s_ml[warp + k * A.join_heads].x);
  const float ref = finite_or_zero(top), f0 = ex2_approx(mx - ref);
  mx = top;
  l *= f0;
  scale4(x, f0);
  for (int k = 1; k < parts; ++k) {
    const float2 ml = s_ml[warp + k * A.join_heads];
    const float f = ex2_approx(ml.x - ref);
    l += f * ml.y;
    add4(x, f, reinterpret_cast<const float4*>(s_x[warp + k * A.join_heads])[lane]);
  }
  T* out = reinterpret_cast<T*>(A.out + b * A.o_b + (head0 + i) * A.o_h) + 4 * lane;
  out[0] = DT<T>::from_f(l == 0.f ? 0.f : x.x / l);
  out[1] = DT<T>::from_f(l == 0.f ? 0.f : x.y / l);
  out[2] = DT<T>::from_f(l == 0.f ? 0.f : x.z / l);
  out[3] = DT<T>::from_f(l == 0.f ? 0.f : x.w / l);
  if (A.lse && lane == 0) A.lse[(int64_t)b * A.hq + head0 + i] = l == 0.f ? -INFINITY : (mx + log2f(l)) * kLn2;
}

}  // namespace fpb
