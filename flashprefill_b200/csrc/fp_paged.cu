// Paged key/value cache: writing rows into it and reading a cached prefix back.
//
// A cache is (pages, page_size, kv_heads, 128) with any page / token / head strides that are multiples of 16 bytes, held
// as the 16-bit type of the rows or as e4m3 codes with one fp32 scale for each (token, head):
//
//   amax  = max(max_d |x_d|, 2^-100)          (the floor keeps a row of zeros, or of denormals, free of 0 / 0)
//   scale = amax / 448,  code_d = e4m3(x_d * (448 / amax)),  read back as code_d * scale rounded to 16 bits
//
// amax is found on the 16-bit patterns with the sign cleared: their integer order is the order of the magnitudes with inf
// and NaN on top, so a row that holds either gets a scale of inf or NaN and reads back as NaN throughout (fmaxf would drop
// the NaN).  The rounding to e4m3 is the purpose of the type: half the bytes, an error of at most 2^-4 of each value.
//
// Both kernels are bound by HBM: each byte moves once, in 16-byte pieces, and one (token, head) row of K and of V is the
// work of 16 lanes (16-bit cache) or 8 lanes (e4m3: 16 elements a lane, so that amax takes three shuffles and the codes of
// a lane are one 16-byte store).
#include "fp_common.cuh"

namespace fpb {

// Error bits of the paged kernels (they have no workspace): sticky, read and cleared by fpb_paged_read_device_error.
__device__ uint32_t g_paged_err;

enum : uint32_t {
  kErrBadPage = 1u << 4,    // a slot or a page-table entry outside the cache
  kErrBadLength = 1u << 5,  // a sequence length outside [0, room]
};

struct PagedCache {
  uint8_t *k, *v;             // codes or 16-bit values
  float *k_scale, *v_scale;   // e4m3 only
  int64_t s_page, s_tok, s_head;     // bytes
  int64_t ss_page, ss_tok, ss_head;  // scale strides in elements
  int num_pages, page_size;
};

// Longest sequence: token indices and their rounding up to whole tiles stay in 32 bits.
constexpr int64_t kPagedMaxLen = (int64_t(1) << 31) - 1024;
constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;  // 2^-100

// Two e4m3 codes (low byte first) as fp16 pair, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two));
  return r;
}
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// max over the 16-bit magnitudes of a packed pair, lane by lane
__device__ __forceinline__ uint32_t absmax2(uint32_t m, uint32_t x) { return __vmaxu2(m, x & 0x7FFF7FFFu); }

__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }

// ------------------------------------------------------------------ write
struct KvWriteArgs {
  PagedCache C;
  const uint8_t *k, *v;
  int64_t ks_tok, ks_head, vs_tok, vs_head;  // bytes
  const void* slots;
  int slots64;
  unsigned rows, hk;  // tokens * kv heads
};

__device__ __forceinline__ int64_t load_slot(const KvWriteArgs& A, unsigned tok) {
  return A.slots64 ? __ldg(static_cast<const long long*>(A.slots) + tok)
                   : (int64_t)__ldg(static_cast<const int*>(A.slots) + tok);
}

// (page, offset) of a slot; false for padding (negative) and for a slot outside the cache, which is reported.
__device__ __forceinline__ bool decode_slot(const PagedCache& C, int64_t slot, int64_t& page, int& at) {
  if (slot < 0) return false;
  if (slot >= (int64_t)C.num_pages * C.page_size) {
    raise_error(&g_paged_err, kErrBadPage);
    return false;
  }
  page = slot / C.page_size;
  at = (int)(slot - page * C.page_size);
  return true;
}

__global__ void __launch_bounds__(256) kv_write_copy_kernel(const KvWriteArgs A) {
  const unsigned row = blockIdx.x * 16u + threadIdx.x / 16u, c = threadIdx.x % 16u;
  if (row >= A.rows) return;
  const unsigned tok = row / A.hk, h = row - tok * A.hk;
  const uint4 kx = __ldcs(reinterpret_cast<const uint4*>(A.k + tok * A.ks_tok + h * A.ks_head) + c);
  const uint4 vx = __ldcs(reinterpret_cast<const uint4*>(A.v + tok * A.vs_tok + h * A.vs_head) + c);
  int64_t page;
  int at;
  if (!decode_slot(A.C, load_slot(A, tok), page, at)) return;
  const int64_t off = page * A.C.s_page + at * A.C.s_tok + h * A.C.s_head;
  reinterpret_cast<uint4*>(A.C.k + off)[c] = kx;
  reinterpret_cast<uint4*>(A.C.v + off)[c] = vx;
}

// One lane's 16 elements of a row: amax over the 8 lanes of the row, then codes and (first lane) the scale.
template <typename T>
__device__ __forceinline__ void quantise_row(const uint4 (&x)[2], uint8_t* dst, float* scale, unsigned c, unsigned mask) {
  const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = absmax2(m, w[i]);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(mask, m, o));
  m = max(m & 0xFFFFu, m >> 16);
  float amax = DT<T>::lo(m);
  amax = amax < kAmaxFloor ? kAmaxFloor : amax;  // NaN stays NaN
  const float inv = __fdiv_rn(kE4m3Max, amax);
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out[i] = f32x2_to_e4m3x2(DT<T>::lo(w[2 * i]) * inv, DT<T>::hi(w[2 * i]) * inv) |
             f32x2_to_e4m3x2(DT<T>::lo(w[2 * i + 1]) * inv, DT<T>::hi(w[2 * i + 1]) * inv) << 16;
  reinterpret_cast<uint4*>(dst)[c] = make_uint4(out[0], out[1], out[2], out[3]);
  if (c == 0) *scale = __fdiv_rn(amax, kE4m3Max);
}

template <typename T>
__global__ void __launch_bounds__(256) kv_write_e4m3_kernel(const KvWriteArgs A) {
  const unsigned row = blockIdx.x * 32u + threadIdx.x / 8u, c = threadIdx.x % 8u;
  if (row >= A.rows) return;
  const unsigned tok = row / A.hk, h = row - tok * A.hk;
  const uint4* kp = reinterpret_cast<const uint4*>(A.k + tok * A.ks_tok + h * A.ks_head) + 2 * c;
  const uint4* vp = reinterpret_cast<const uint4*>(A.v + tok * A.vs_tok + h * A.vs_head) + 2 * c;
  const uint4 kx[2] = {__ldcs(kp), __ldcs(kp + 1)};
  const uint4 vx[2] = {__ldcs(vp), __ldcs(vp + 1)};
  int64_t page;
  int at;
  if (!decode_slot(A.C, load_slot(A, tok), page, at)) return;  // the same for all 8 lanes of a row
  const unsigned mask = 0xFFu << (threadIdx.x & 24u);
  const int64_t off = page * A.C.s_page + at * A.C.s_tok + h * A.C.s_head;
  const int64_t soff = page * A.C.ss_page + at * A.C.ss_tok + h * A.C.ss_head;
  quantise_row<T>(kx, A.C.k + off, A.C.k_scale + soff, c, mask);
  quantise_row<T>(vx, A.C.v + off, A.C.v_scale + soff, c, mask);
}

// ------------------------------------------------------------------ read
struct KvReadArgs {
  PagedCache C;
  const int* page_table;
  int64_t table_stride;
  int max_pages;
  const int* seq_lens;
  int out_len, hk;
  uint8_t *k, *v;
  int64_t ks_b, ks_tok, ks_head, vs_b, vs_tok, vs_head;  // bytes
};

// Cached row (b, s, h) of the item `row` = s * hk + h; false where there is none to copy.
__device__ __forceinline__ bool read_row(const KvReadArgs& A, unsigned row, int b, int& s, int& h, int64_t& page, int& at) {
  s = row / (unsigned)A.hk;
  h = row - s * A.hk;
  const int len = __ldg(A.seq_lens + b);
  const int64_t room = min((int64_t)A.max_pages * A.C.page_size, (int64_t)A.out_len);
  if (len < 0 || len > room) {
    raise_error(&g_paged_err, kErrBadLength);
    return false;
  }
  if (s >= len) return false;
  const int p = s / A.C.page_size;
  at = s - p * A.C.page_size;
  page = __ldg(A.page_table + b * A.table_stride + p);
  if (page < 0 || page >= A.C.num_pages) {
    raise_error(&g_paged_err, kErrBadPage);
    return false;
  }
  return true;
}

__global__ void __launch_bounds__(256) kv_read_copy_kernel(const KvReadArgs A) {
  const unsigned row = blockIdx.x * 16u + threadIdx.x / 16u, c = threadIdx.x % 16u;
  const int b = blockIdx.y;
  if (row >= (unsigned)A.out_len * (unsigned)A.hk) return;
  int s, h, at;
  int64_t page;
  if (!read_row(A, row, b, s, h, page, at)) return;
  const int64_t off = page * A.C.s_page + at * A.C.s_tok + h * A.C.s_head;
  const uint4 kx = __ldg(reinterpret_cast<const uint4*>(A.C.k + off) + c);
  const uint4 vx = __ldg(reinterpret_cast<const uint4*>(A.C.v + off) + c);
  reinterpret_cast<uint4*>(A.k + b * A.ks_b + s * A.ks_tok + h * A.ks_head)[c] = kx;
  reinterpret_cast<uint4*>(A.v + b * A.vs_b + s * A.vs_tok + h * A.vs_head)[c] = vx;
}

template <typename T>
__device__ __forceinline__ void dequantise_row(uint4 x, float scale, uint4* dst) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t out[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t p = e4m3x2_to_f16x2(i & 1 ? w[i / 2] >> 16 : w[i / 2]);
    out[i] = DT<T>::pack(DT<__half>::lo(p) * scale, DT<__half>::hi(p) * scale);
  }
  dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
  dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
}

template <typename T>
__global__ void __launch_bounds__(256) kv_read_e4m3_kernel(const KvReadArgs A) {
  const unsigned row = blockIdx.x * 32u + threadIdx.x / 8u, c = threadIdx.x % 8u;
  const int b = blockIdx.y;
  if (row >= (unsigned)A.out_len * (unsigned)A.hk) return;
  int s, h, at;
  int64_t page;
  if (!read_row(A, row, b, s, h, page, at)) return;
  const int64_t off = page * A.C.s_page + at * A.C.s_tok + h * A.C.s_head;
  const int64_t soff = page * A.C.ss_page + at * A.C.ss_tok + h * A.C.ss_head;
  const uint4 kx = __ldg(reinterpret_cast<const uint4*>(A.C.k + off) + c);
  const uint4 vx = __ldg(reinterpret_cast<const uint4*>(A.C.v + off) + c);
  const float ks = __ldg(A.C.k_scale + soff), vs = __ldg(A.C.v_scale + soff);
  dequantise_row<T>(kx, ks, reinterpret_cast<uint4*>(A.k + b * A.ks_b + s * A.ks_tok + h * A.ks_head) + 2 * c);
  dequantise_row<T>(vx, vs, reinterpret_cast<uint4*>(A.v + b * A.vs_b + s * A.vs_tok + h * A.vs_head) + 2 * c);
}

__global__ void paged_clear_err_kernel(uint32_t bits) { atomicAnd(&g_paged_err, ~bits); }

}  // namespace fpb
