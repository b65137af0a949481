// Attention of one new token for each sequence over its pages of the cache (fp_paged.cu), split over the cache's length
// and joined.
//
//   s_j = sm_scale * q . k_j,   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   lse = m + log sum_j exp(s_j - m)
//
// for every sequence b and query head, j over the sequence's seq_lens[b] cached tokens; the G = hq / hk query heads of a
// KV head share its rows.  Each cached byte is read once and meets 2 G flops (2-byte cache), so the operator is bound by
// HBM; the arithmetic only has to stay out of the way.
//
// Work.  An item is (sequence, KV head, group of query heads: all G up to 8 NT, equal groups above that).  All items' tokens, cut into units of
// kWarps * TT tokens, form one line, and each of a fixed number of CTAs takes an equal stretch of it, so ragged batches
// and single long sequences load the GPU alike, whatever the lengths (they are read on the device: no host copy, and a
// captured graph serves any lengths).  A stretch that covers a whole item writes its output; an item cut by a CTA border
// leaves unnormalised sums and their maxima in the workspace, which a second kernel (programmatic dependent launch)
// joins in the order of the tokens: no atomics, the same bits on every run.  The second kernel is not launched where
// no item can have two units.
//
// A warp works alone on its own tiles of TT tokens (16 of a 16-bit cache, 32 of e4m3: 4 KB of K and of V each way) through
// a ring of kStages tiles filled by 16-byte cp.async, so loads are in flight all the time without block-wide barriers;
// warps meet once an item.  Rows behind the end, or on a page that is not in the cache, are filled with zeros and their
// scores set to -inf: stale values there never reach the sums.
//
// Tensor cores.  S^T = K Q^T with the tokens as the 16 rows and 8 heads as the columns of mma.m16n8k16; out^T = V^T P^T
// with the channels as rows.  The small side of both products is the 8-wide one, so G <= 8 heads cost one pass where
// tcgen05's least tile would be mostly padding, and the operands need no staging beyond the ring.
//   * Scores, maxima, sums and outputs stay in fp32 registers; running maximum, rescaled only when it moves.
//   * bf16 V: P is split into two bf16 parts (the value and its remainder) and multiplied twice: one bf16 P would leave
//     errors as large as the output's own rounding.
//   * fp16 V: P is scaled by 2^15 (as the row sum is, so it cancels), which keeps weights down to 2^-29 of the largest in
//     fp16's normal range.
//   * e4m3: codes widen to fp16 exactly; q is scaled by a power of two to fit fp16; the token's K scale multiplies its
//     score and its V scale its weight, relative to the largest V scale so far (a power-free running reference like the
//     maximum), so weights stay at most 2^15.
#include <type_traits>

#include "fp_common.cuh"

namespace fpb {

constexpr int kDecWarps = 4;
constexpr int kDecStages = 3;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kDecTileBytes = 4096;  // one warp's tile of K or of V
constexpr int kDecRingBytes = kDecStages * 2 * kDecTileBytes;
constexpr int kDecSmemBytes = kDecWarps * kDecRingBytes;
constexpr int kDecCtasPerSm = 2;
constexpr int kDecMaxCtas = 512;   // bound of the workspace
constexpr int kJoinThreads = 512;
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
  int max_pages, batch, hq, hk;
  int G, ngroups, nh;                // query heads of a KV head, groups of them, heads of a group (the last may have fewer)
  float c;                           // sm_scale * log2(e)
  int4* desc;                        // per CTA: {b, KV head * groups + group, partials, 0} of the item it begins and does not end
  float* part;                       // [2 * CTA + slot][nh][128]
  float2* ml;                        // [2 * CTA + slot][nh] {maximum (log2 units), sum}
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// Tokens of sequence b; a length outside [0, room] is reported and counts as 0.
__device__ __forceinline__ int seq_len_of(const DecodeArgs& A, int b) {
  const int len = __ldg(A.seq_lens + b);
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
  static constexpr bool kSplitP = DT<MT>::is_bf16;
  static constexpr float kShift = kSplitP ? 0.f : 15.f;  // log2 of the factor of P and l

  uint32_t ring;  // shared address of this warp's ring
  int lane;
  uint32_t qf[NT][8][2];      // q as the B operand
  float qc[NT][2];            // factor of this thread's two columns (heads 2t, 2t + 1)
  float o[NT][8][4];          // out^T: 16 channels x 8 heads a tile
  float m[NT][2], l[NT][2];   // running maximum and this thread's share of the sum
  float vref;                 // e4m3: largest V scale so far

  __device__ __forceinline__ void load_q(const DecodeArgs& A, const uint8_t* q, int heads) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool ok = n * 8 + g < heads;
      const uint8_t* row = q + (n * 8 + g) * A.q_h;
      float f = 1.f;
      if constexpr (!kE4m3) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          qf[n][k][0] = ok ? __ldg(reinterpret_cast<const uint32_t*>(row + 32 * k + 4 * t)) : 0u;
          qf[n][k][1] = ok ? __ldg(reinterpret_cast<const uint32_t*>(row + 32 * k + 4 * t + 16)) : 0u;
        }
      } else {
        // an e4m3 row gives a thread elements 4t .. 4t+3 of each 16: they take the places 2t, 2t+1, 2t+8, 2t+9 of the
        // product's inner dimension, in q as in K
        uint32_t mx = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint2 x = ok ? __ldg(reinterpret_cast<const uint2*>(row + 32 * k + 8 * t)) : make_uint2(0u, 0u);
          qf[n][k][0] = x.x;
          qf[n][k][1] = x.y;
          mx = absmax2(absmax2(mx, x.x), x.y);
        }
        if constexpr (DT<T>::is_bf16) {
          mx = max(mx & 0xFFFFu, mx >> 16);
          mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          // power of two that brings the row's largest magnitude to [1, 2); inf and NaN pass as they are
          int e = (int)(mx >> 7) - 127;
          e = max(-120, min(e, 120));
          const float down = exp2i(-e);
          f = exp2i(e);
#pragma unroll
          for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              qf[n][k][j] = DT<__half>::pack(DT<T>::lo(qf[n][k][j]) * down, DT<T>::hi(qf[n][k][j]) * down);
        }
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
    vref = 1.1754943508222875e-38f;
  }

  // Starts the copies of tokens [tok, tok + TT) below `end` into ring slot `stage`; kvalid: bit r set where row r is there;
  // ks, vs: this lane's token's scales.
  __device__ __forceinline__ void issue(const DecodeArgs& A, const int* table, int64_t head_off, int64_t scale_off, int tok,
                                        int end, int stage, uint32_t& kvalid, float& ks, float& vs) {
    const int r0 = lane % TT, my = tok + r0;
    int64_t off = -1;
    ks = vs = 0.f;
    if (my < end) {
      const int p = my / A.C.page_size, at = my - p * A.C.page_size;
      const int page = __ldg(table + p);
      if (page >= 0 && page < A.C.num_pages) {
        off = (int64_t)page * A.C.s_page + (int64_t)at * A.C.s_tok;
        if constexpr (kE4m3) {
          const int64_t so = (int64_t)page * A.C.ss_page + (int64_t)at * A.C.ss_tok + scale_off;
          ks = __ldg(A.C.k_scale + so);
          vs = __ldg(A.C.v_scale + so);
        }
      } else {
        raise_error(&g_paged_err, kErrBadPage);
      }
    }
    kvalid = __ballot_sync(0xffffffffu, off >= 0);
    const uint32_t kd = ring + stage * 2 * kDecTileBytes, vd = kd + kDecTileBytes;
    const int ch = lane % kChunks;
    constexpr int kRowsPer = 32 / kChunks;
#pragma unroll
    for (int i = 0; i < TT / kRowsPer; ++i) {
      const int r = i * kRowsPer + lane / kChunks;
      const int64_t ro = __shfl_sync(0xffffffffu, off, r);
      const uint32_t d = r * kRowBytes + ((ch ^ (r & 7)) << 4);
      const int64_t so = ro < 0 ? 0 : ro + head_off + ch * 16;
      cp_async16(kd + d, A.C.k + so, ro < 0 ? 0 : 16);
      cp_async16(vd + d, A.C.v + so, ro < 0 ? 0 : 16);
    }
  }

  __device__ __forceinline__ void consume(int stage, uint32_t kvalid, float ks, float vs) {
    const uint32_t kd = ring + stage * 2 * kDecTileBytes, vd = kd + kDecTileBytes;
    const int g = lane >> 2;
    float s[NT][MTILES][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][i][j] = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t a[4];
      if constexpr (!kE4m3) {
        const int r = lane & 15, ch = 2 * k + (lane >> 4);
        ldsm4(a, kd + r * kRowBytes + ((ch ^ (r & 7)) << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<MT>(s[n][0], a[0], a[1], a[2], a[3], qf[n][k][0], qf[n][k][1]);
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
    // row factors of this thread's tokens g, g + 8 (+ 16 i)
    float kf[MTILES][2], vf[MTILES][2];
    float vcorr = 1.f;
    if constexpr (kE4m3) {
      const float vmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vs)));
      const float vnew = vmax > vref || vmax != vmax ? vmax : vref;
      vcorr = vref / vnew;
      vref = vnew;
      const float vw = vs / vnew;
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          kf[i][j] = __shfl_sync(0xffffffffu, ks, 16 * i + 8 * j + g);
          vf[i][j] = __shfl_sync(0xffffffffu, vw, 16 * i + 8 * j + g);
        }
    }
    bool moved = vcorr != 1.f;
    float corr[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // the column (head) 2t + j
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < MTILES; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x = s[n][i][2 * h + j] * qc[n][j];
            if constexpr (kE4m3) x *= kf[i][h];
            x = (kvalid >> (16 * i + 8 * h + g)) & 1u ? x : -INFINITY;
            s[n][i][2 * h + j] = x;
            mx = fmaxf(mx, x);
          }
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float mn = fmaxf(m[n][j], mx), ref = finite_or_zero(mn);
        moved |= mn != m[n][j];
        const float cr = ex2_approx(m[n][j] - ref);
        m[n][j] = mn;
        l[n][j] *= cr;
        corr[n][j] = cr * vcorr;
#pragma unroll
        for (int i = 0; i < MTILES; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float p = ex2_approx(s[n][i][2 * h + j] - (ref - kShift));
            l[n][j] += p;
            s[n][i][2 * h + j] = kE4m3 ? p * vf[i][h] : p;
          }
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][i][j] *= corr[n][j & 1];
    }
    uint32_t pb[NT][MTILES][2], pl[NT][MTILES][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x0 = s[n][i][2 * h], x1 = s[n][i][2 * h + 1];
          const uint32_t hi = DT<MT>::pack(x0, x1);
          pb[n][i][h] = transpose8x8(hi);
          if constexpr (kSplitP) pl[n][i][h] = transpose8x8(DT<MT>::pack(x0 - DT<MT>::lo(hi), x1 - DT<MT>::hi(hi)));
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
          for (int n = 0; n < NT; ++n) mma16816<MT>(o[n][i], a0, a1, a2, a3, pb[n][k][0], pb[n][k][1]);
        }
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
        if (g == 0) sml[h] = make_float2(m[n][j] - kShift, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = kE4m3 ? vref : 1.f;
          const int d0 = 16 * i + (kE4m3 ? 2 * g : g), d1 = 16 * i + (kE4m3 ? 2 * g + 1 : g + 8);
          so[h * 132 + d0] = o[n][i][j] * f;
          so[h * 132 + d1] = o[n][i][2 + j] * f;
        }
      }
  }
};

template <typename T, bool kE4m3, int NT>
__global__ void __launch_bounds__(kDecThreads, kDecCtasPerSm) paged_decode_kernel(const DecodeArgs A) {
  using W = DecodeWarp<T, kE4m3, NT>;
  constexpr int kUnit = kDecWarps * W::TT;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 s_ml[kDecWarps][8 * NT];
  __shared__ int64_t s_scan[kDecWarps];
  __shared__ int64_t s_start[2];
  static_assert(8 * NT * 132 * 4 <= kDecRingBytes, "a warp's sums fit its ring");

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int HH = A.hk * A.ngroups;

  // ---- this CTA's stretch: prefix sums of the sequences' units (a sequence without tokens has one, empty)
  const int per = (A.batch + kDecThreads - 1) / kDecThreads;
  const int b_lo = min(tid * per, A.batch), b_hi = min(b_lo + per, A.batch);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += max(1, (seq_len_of(A, b) + kUnit - 1) / kUnit);
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += x;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  int64_t total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kDecWarps; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  incl += before;
  total *= HH;
  const int64_t ctas = min((int64_t)gridDim.x, total);
  if (A.desc && tid == 0) A.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
  if ((int64_t)blockIdx.x >= ctas) return;
  int64_t t = (int64_t)blockIdx.x * total / ctas;
  const int64_t t_end = ((int64_t)blockIdx.x + 1) * total / ctas;
  {
    int64_t base = (incl - mine) * HH;
    if (base <= t && t < incl * HH) {  // one thread
      int b = b_lo;
      while (true) {
        const int64_t n = (int64_t)max(1, (seq_len_of(A, b) + kUnit - 1) / kUnit) * HH;
        if (t < base + n) break;
        base += n;
        ++b;
      }
      s_start[0] = b;
      s_start[1] = base;
    }
  }
  __syncthreads();
  int b = (int)s_start[0];
  int len = seq_len_of(A, b);
  int units = max(1, (len + kUnit - 1) / kUnit);
  int hh = (int)((t - s_start[1]) / units);
  int u = (int)((t - s_start[1]) - (int64_t)hh * units);

  W w;
  w.lane = lane;
  w.ring = smem_u32(smem) + warp * kDecRingBytes;
  float* const so = reinterpret_cast<float*>(smem + warp * kDecRingBytes);

  while (t < t_end) {
    const int u_end = (int)min((int64_t)units, u + (t_end - t));
    const int h = hh / A.ngroups, grp = hh - h * A.ngroups;
    const int head0 = h * A.G + grp * A.nh, heads = min(A.nh, A.G - grp * A.nh);
    const int tok0 = u * kUnit, end = min(len, u_end * kUnit);
    const int* table = A.page_table + b * A.table_stride;
    const int64_t head_off = h * A.C.s_head, scale_off = h * A.C.ss_head;
    const int tiles = (end - tok0 + W::TT - 1) / W::TT;           // of the stretch (<= 0: none)
    const int n = tiles > warp ? (tiles - warp + kDecWarps - 1) / kDecWarps : 0;  // of this warp

    uint32_t valid[kDecStages];
    float ks[kDecStages], vs[kDecStages];
#pragma unroll
    for (int i = 0; i < kDecStages - 1; ++i) {
      if (i < n) w.issue(A, table, head_off, scale_off, tok0 + (i * kDecWarps + warp) * W::TT, end, i, valid[i], ks[i], vs[i]);
      cp_async_commit();
    }
    w.load_q(A, A.q + b * A.q_b + head0 * A.q_h, heads);
    w.reset();
    for (int i0 = 0; i0 < n; i0 += kDecStages) {
#pragma unroll
      for (int j = 0; j < kDecStages; ++j) {
        if (i0 + j < n) {
          cp_async_wait<kDecStages - 2>();
          __syncwarp();
          const int nx = i0 + j + kDecStages - 1;
          constexpr int kBack = kDecStages - 1;
          const int st = (j + kBack) % kDecStages;
          if (nx < n)
            w.issue(A, table, head_off, scale_off, tok0 + (nx * kDecWarps + warp) * W::TT, end, st, valid[st], ks[st], vs[st]);
          cp_async_commit();
          w.consume(j, valid[j], ks[j], vs[j]);
          __syncwarp();
        }
      }
    }
    cp_async_wait<0>();
    __syncwarp();
    w.store(so, s_ml[warp]);
    __syncthreads();

    const bool whole = u == 0 && u_end == units;
    const int slot = 2 * blockIdx.x + (u == 0 ? 1 : 0);
    for (int i = 0; i < heads; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < kDecWarps; ++k) mx = fmaxf(mx, s_ml[k][i].x);
      const float ref = finite_or_zero(mx);
      float l = 0.f, x = 0.f;
#pragma unroll
      for (int k = 0; k < kDecWarps; ++k) {
        const float f = ex2_approx(s_ml[k][i].x - ref);
        l += f * s_ml[k][i].y;
        x += f * reinterpret_cast<const float*>(smem + k * kDecRingBytes)[i * 132 + tid];
      }
      if (whole) {
        const int head = head0 + i;
        reinterpret_cast<T*>(A.out + b * A.o_b + head * A.o_h)[tid] = DT<T>::from_f(l == 0.f ? 0.f : x / l);
        if (A.lse && tid == 0) A.lse[(int64_t)b * A.hq + head] = l == 0.f ? -INFINITY : (mx + log2f(l)) * kLn2;
      } else {
        A.part[((int64_t)slot * A.nh + i) * kHeadDim + tid] = x;
        if (tid == 0) A.ml[(int64_t)slot * A.nh + i] = make_float2(mx, l);
      }
    }
    if (!whole && u == 0 && tid == 0) {
      const int64_t last = t + units - 1;  // unit of the item's end; its CTA
      const int64_t c1 = ((last + 1) * ctas - 1) / total;
      A.desc[blockIdx.x] = make_int4(b, hh, (int)(c1 - blockIdx.x) + 1, 0);
    }
    __syncthreads();

    t += u_end - u;
    u = 0;
    if (++hh == HH) {
      hh = 0;
      if (++b < A.batch) {
        len = seq_len_of(A, b);
        units = max(1, (len + kUnit - 1) / kUnit);
      }
    }
  }
}

// Joins the partial sums of the item that CTA blockIdx.x of the first kernel began and did not end.  A warp takes one head
// and every parts-th partial (all maxima first, then the weighted sums, four channels a lane); the parts meet in shared
// memory.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_decode_join_kernel(const DecodeArgs A) {
  __shared__ float s_x[kJoinThreads / 32][kHeadDim];
  __shared__ float s_l[kJoinThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 d = A.desc[blockIdx.x];
  const int n = d.z;
  if (n == 0) return;
  const int b = d.x, h = d.y / A.ngroups, grp = d.y - h * A.ngroups;
  const int head0 = h * A.G + grp * A.nh, heads = min(A.nh, A.G - grp * A.nh);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kJoinThreads / 32;
  const int parts = kWarps / heads;  // heads <= 16
  const int i = warp % heads, part = warp / heads;
  auto slot = [&](int k) { return (int64_t)(2 * (blockIdx.x + k) + (k == 0 ? 1 : 0)) * A.nh + i; };
  float mx = -INFINITY;
  for (int k = lane; k < n; k += 32) mx = fmaxf(mx, A.ml[slot(k)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float ref = finite_or_zero(mx);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  if (part < parts) {
#pragma unroll 8
    for (int k = part; k < n; k += parts) {
      const float2 ml = A.ml[slot(k)];
      const float4 p = reinterpret_cast<const float4*>(A.part + slot(k) * kHeadDim)[lane];
      const float f = ex2_approx(ml.x - ref);
      l += f * ml.y;
      x.x += f * p.x;
      x.y += f * p.y;
      x.z += f * p.z;
      x.w += f * p.w;
    }
    reinterpret_cast<float4*>(s_x[warp])[lane] = x;
    if (lane == 0) s_l[warp] = l;
  }
  __syncthreads();
  if (part != 0) return;
  for (int k = 1; k < parts; ++k) {
    const float4 p = reinterpret_cast<const float4*>(s_x[warp + k * heads])[lane];
    l += s_l[warp + k * heads];
    x.x += p.x;
    x.y += p.y;
    x.z += p.z;
    x.w += p.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = reinterpret_cast<T*>(A.out + b * A.o_b + (head0 + i) * A.o_h) + 4 * lane;
  if (l == 0.f) x = make_float4(0.f, 0.f, 0.f, 0.f);
  out[0] = DT<T>::from_f(x.x * inv);
  out[1] = DT<T>::from_f(x.y * inv);
  out[2] = DT<T>::from_f(x.z * inv);
  out[3] = DT<T>::from_f(x.w * inv);
  if (A.lse && lane == 0) A.lse[(int64_t)b * A.hq + head0 + i] = l == 0.f ? -INFINITY : (mx + log2f(l)) * kLn2;
}

}  // namespace fpb
