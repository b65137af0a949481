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
// the NaN).  The rounding to e4m3 is the purpose of the type: half the bytes, an error of at most 2^-4 of each value or 2^-10 of
// the row's scale, whichever is larger.
//
// Both kernels are bound by HBM: each byte moves once, a (token, head) row of K and of V by a group of lanes.  Reading and
// copying take 16 lanes of 16 bytes a row; quantising takes 8 lanes of 16 elements, because the work of a row that does not
// shrink with its elements (amax over the lanes, the division, the addresses) would bound it with 16 lanes (131072 tokens of
// 8 heads, bf16 to e4m3: 177 us against 134).  Where a read is large enough to fill the GPU all the same and 4 divides
// page_size, the lanes take 4 tokens of a head: one table entry and one division for all, and their loads under way together (the same
// tokens read back: 127 us, 140 token by token).  As rows are read once, loads that leave the caches first might seem right, but
// they were written just before, and are still in L2 in the calls that matter (4099 tokens of 2 heads to e4m3: 2.5 us, 2.9 so).
// Of the measured 6.54 TB/s at 131072 tokens of 8 heads: copying 101%, quantising 94% (57% of the issue slots), reading e4m3 97%.
#include "fp_common.cuh"

namespace fpb {

// Error bits of the paged kernels (they have no workspace): sticky, read and cleared by fpb_paged_read_device_error.
__device__ uint32_t g_paged_err;

enum : uint32_t {
  kErrBadPage = 1u << 4,    // a slot or a page-table entry outside the cache
  kErrBadLength = 1u << 5,  // a sequence length outside [0, room]
};

// x / d for 0 <= x < 2^31: mul exceeds 2^shift / d by at most one, shift = 31 + ceil(log2 d).
struct FastDiv {
  unsigned mul;
  int shift;
  __device__ __forceinline__ unsigned operator()(unsigned x) const { return (unsigned)(((uint64_t)x * mul) >> shift); }
};

// Element (a, token, head) of a tensor whose three strides are in 16-byte pieces (rows) or in elements (scales).
struct Pitch {
  unsigned outer, tok, head;
  __device__ __forceinline__ uint64_t at(unsigned a, unsigned t, unsigned h) const {
    return (uint64_t)a * outer + (uint64_t)t * tok + (uint64_t)h * head;
  }
};

struct PagedCache {
  uint8_t *k, *v;            // codes or 16-bit values
  float *k_scale, *v_scale;  // e4m3 only
  Pitch rows, scales;        // outer: page
  int num_pages, page_size;
  FastDiv page_of;           // token -> index into its sequence's table; slot -> page
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
// The kernels of the paged cache are short and follow one another (write, decode, join, the next layer's write ...), so each
// is launched with programmatic stream serialisation, which prepares its launch while its predecessor still runs, and waits
// here, before it touches memory, until all that came before it on the stream is complete and visible (1 x 500 tokens
// decode: 6.2 us a call without, 4.6 with).  What it then reads may have been written while it was already launched, so its
// loads are ordinary ones: the read-only path (__ldg) asks for memory that no one writes for as long as the kernel lives, and
// the compiler may move such loads, even in front of the wait (without them 131072 tokens to e4m3 take 126.2 us, 125.5 with;
// 1 x 500 tokens decode 4.4, 4.5 with).
__device__ __forceinline__ void await_stream() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// (a0, a1) * b, two products in one instruction
__device__ __forceinline__ float2 mul2(float a0, float a1, float b) {
  float2 d;
  asm("{\n .reg .b64 ra, rb, rd;\n mov.b64 ra, {%2, %3};\n mov.b64 rb, {%4, %4};\n mul.rn.f32x2 rd, ra, rb;\n"
      " mov.b64 {%0, %1}, rd;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a0), "f"(a1), "f"(b));
  return d;
}
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float2 x) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(x.y), "f"(x.x));
  return r;
}

// max over the 16-bit magnitudes of a packed pair, lane by lane
__device__ __forceinline__ uint32_t absmax2(uint32_t m, uint32_t x) { return __vmaxu2(m, x & 0x7FFF7FFFu); }

__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }

// ------------------------------------------------------------------ write
struct KvWriteArgs {
  PagedCache C;
  const uint8_t *k, *v;
  Pitch kp, vp;  // outer unused
  const void* slots;
  int slots64;
  unsigned rows, hk;  // tokens * kv heads
  FastDiv token_of;   // row -> token
};

__device__ __forceinline__ int64_t load_slot(const KvWriteArgs& A, unsigned tok) {
  return A.slots64 ? static_cast<const int64_t*>(A.slots)[tok] : static_cast<const int*>(A.slots)[tok];
}

// (page, offset) of a slot; false for padding (negative) and for a slot outside the cache, which is reported.
__device__ __forceinline__ bool decode_slot(const PagedCache& C, int64_t slot, int64_t& page, int& at) {
  if (slot < 0) return false;
  if (slot >= (int64_t)C.num_pages * C.page_size) {
    raise_error(&g_paged_err, kErrBadPage);
    return false;
  }
  page = slot < (int64_t(1) << 31) ? (int64_t)C.page_of((unsigned)slot) : slot / C.page_size;
  at = (int)(slot - page * C.page_size);
  return true;
}

constexpr int kRowThreads = 256;
constexpr int row_lanes(bool quantise) { return quantise ? 8 : 16; }                      // lanes of a row
constexpr int block_rows(bool quantise) { return kRowThreads / row_lanes(quantise); }  // rows of a block at a time

// One lane's 16 elements of a row: amax over the row's 8 lanes, then the codes and (first lane) the scale.
template <typename T>
__device__ __forceinline__ void quantise_row(const uint4 (&x)[2], uint4* dst, float* scale, unsigned c, unsigned mask) {
  const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = absmax2(m, w[i]);
#pragma unroll
  for (int o = 1; o < row_lanes(true); o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(mask, m, o));
  m = max(m & 0xFFFFu, m >> 16);
  float amax = DT<T>::lo(m);
  amax = amax < kAmaxFloor ? kAmaxFloor : amax;  // NaN stays NaN
  const float inv = __fdiv_rn(kE4m3Max, amax);
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out[i] = f32x2_to_e4m3x2(mul2(DT<T>::lo(w[2 * i]), DT<T>::hi(w[2 * i]), inv)) |
             f32x2_to_e4m3x2(mul2(DT<T>::lo(w[2 * i + 1]), DT<T>::hi(w[2 * i + 1]), inv)) << 16;
  dst[c] = make_uint4(out[0], out[1], out[2], out[3]);
  if (c == 0) *scale = __fdiv_rn(amax, kE4m3Max);
}

// T: type of the rows (a 16-bit cache gets a copy whatever it is).
template <typename T, bool kE4m3>
__global__ void __launch_bounds__(kRowThreads, kE4m3 ? 6 : 8) kv_write_kernel(const KvWriteArgs A) {
  constexpr int kLanes = row_lanes(kE4m3), kPieces = 16 / kLanes;  // 16-byte pieces of a lane
  await_stream();
  const unsigned c = threadIdx.x % kLanes, row = blockIdx.x * block_rows(kE4m3) + threadIdx.x / kLanes;
  if (row >= A.rows) return;
  const unsigned tok = A.token_of(row), h = row - tok * A.hk;
  const int64_t slot = load_slot(A, tok);
  const uint4* kp = reinterpret_cast<const uint4*>(A.k) + A.kp.at(0, tok, h) + c * kPieces;
  const uint4* vp = reinterpret_cast<const uint4*>(A.v) + A.vp.at(0, tok, h) + c * kPieces;
  uint4 kx[kPieces], vx[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) kx[i] = kp[i];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) vx[i] = vp[i];
  int64_t page;
  int at;
  if (!decode_slot(A.C, slot, page, at)) return;  // the same for all lanes of a row
  const uint64_t off = A.C.rows.at((unsigned)page, at, h);
  uint4* ko = reinterpret_cast<uint4*>(A.C.k) + off;
  uint4* vo = reinterpret_cast<uint4*>(A.C.v) + off;
  if constexpr (kE4m3) {
    const unsigned mask = 0xFFu << (threadIdx.x & 24u);
    const uint64_t soff = A.C.scales.at((unsigned)page, at, h);
    quantise_row<T>(kx, ko, A.C.k_scale + soff, c, mask);
    quantise_row<T>(vx, vo, A.C.v_scale + soff, c, mask);
  } else {
    ko[c] = kx[0];
    vo[c] = vx[0];
  }
}

// ------------------------------------------------------------------ read
struct KvReadArgs {
  PagedCache C;
  const int* page_table;
  int64_t table_stride;
  int max_pages;
  const int* seq_lens;
  int out_len, hk;
  FastDiv group_of;  // item / hk
  uint8_t *k, *v;
  Pitch kp, vp;      // outer: sequence
};

template <typename T>
__device__ __forceinline__ uint4 dequantise8(uint2 x, float scale) {
  const uint32_t p[4] = {e4m3x2_to_f16x2(x.x), e4m3x2_to_f16x2(x.x >> 16), e4m3x2_to_f16x2(x.y), e4m3x2_to_f16x2(x.y >> 16)};
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = mul2(DT<__half>::lo(p[i]), DT<__half>::hi(p[i]), scale);
    out[i] = DT<T>::pack(f.x, f.y);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// T: type of the rows (a 16-bit cache is copied whatever it is).  16 lanes take kGroup tokens of one head, all on one page
// (kGroup divides page_size); y: sequence.
template <typename T, bool kE4m3, int kGroup>
__global__ void __launch_bounds__(kRowThreads) kv_read_kernel(const KvReadArgs A) {
  constexpr int kLanes = row_lanes(false);
  await_stream();
  const unsigned c = threadIdx.x % kLanes, item = blockIdx.x * block_rows(false) + threadIdx.x / kLanes;
  const int b = blockIdx.y, len = A.seq_lens[b];
  if (len < 0 || len > min((int64_t)A.max_pages * A.C.page_size, (int64_t)A.out_len)) {
    raise_error(&g_paged_err, kErrBadLength);
    return;
  }
  const int group = A.group_of(item), h = item - group * A.hk, s = group * kGroup, n = len - s;
  if (n <= 0) return;
  const int p = A.C.page_of(s), at = s - p * A.C.page_size;
  const int page = A.page_table[b * A.table_stride + p];
  if ((unsigned)page >= (unsigned)A.C.num_pages) {
    raise_error(&g_paged_err, kErrBadPage);
    return;
  }
  uint4* ko = reinterpret_cast<uint4*>(A.k) + A.kp.at(b, s, h) + c;
  uint4* vo = reinterpret_cast<uint4*>(A.v) + A.vp.at(b, s, h) + c;
  const uint64_t off = A.C.rows.at(page, at, h);
  if constexpr (kE4m3) {
    const uint2* kc = reinterpret_cast<const uint2*>(reinterpret_cast<const uint4*>(A.C.k) + off) + c;
    const uint2* vc = reinterpret_cast<const uint2*>(reinterpret_cast<const uint4*>(A.C.v) + off) + c;
    const uint64_t soff = A.C.scales.at(page, at, h);
    uint2 kx[kGroup], vx[kGroup];
    float ks[kGroup], vs[kGroup];
#pragma unroll
    for (int j = 0; j < kGroup; ++j)
      if (j < n) {
        kx[j] = kc[(uint64_t)j * 2 * A.C.rows.tok];
        vx[j] = vc[(uint64_t)j * 2 * A.C.rows.tok];
        ks[j] = A.C.k_scale[soff + (uint64_t)j * A.C.scales.tok];
        vs[j] = A.C.v_scale[soff + (uint64_t)j * A.C.scales.tok];
      }
#pragma unroll
    for (int j = 0; j < kGroup; ++j)
      if (j < n) {
        ko[(uint64_t)j * A.kp.tok] = dequantise8<T>(kx[j], ks[j]);
        vo[(uint64_t)j * A.vp.tok] = dequantise8<T>(vx[j], vs[j]);
      }
  } else {
    const uint4* kc = reinterpret_cast<const uint4*>(A.C.k) + off + c;
    const uint4* vc = reinterpret_cast<const uint4*>(A.C.v) + off + c;
    uint4 kx[kGroup], vx[kGroup];
#pragma unroll
    for (int j = 0; j < kGroup; ++j)
      if (j < n) {
        kx[j] = kc[(uint64_t)j * A.C.rows.tok];
        vx[j] = vc[(uint64_t)j * A.C.rows.tok];
      }
#pragma unroll
    for (int j = 0; j < kGroup; ++j)
      if (j < n) {
        ko[(uint64_t)j * A.kp.tok] = kx[j];
        vo[(uint64_t)j * A.vp.tok] = vx[j];
      }
  }
}

// Takes the error bits and clears them in one step: a bit that another stream's kernel sets afterwards stays for the next read.
__device__ uint32_t g_paged_taken;
__global__ void paged_take_err_kernel() { g_paged_taken = atomicExch(&g_paged_err, 0u); }

}  // namespace fpb
