// What the paged key/value cache's kernels share: its layout, slot and page arithmetic
// with bounds checks, and e4m3 rows with power-of-two scales.
//
// Layout: each of the two caches is (num_pages, Hkv, page_size, D), a page's inner three
// dimensions contiguous, pages `page_stride` elements apart, so that one head's part of a
// page is one run of page_size * D elements. Scales (e4m3 caches) are contiguous fp32
// (num_pages, Hkv, page_size): one per token and head.
//
// e4m3 rows: the scale of a row is the smallest power of two s (2^-126 at least) with
// max|x| / s <= 448, the largest e4m3 value, and 1 for a row of zeros. Dividing by s is
// exact, so a code is one rounding of x (to nearest, ties to even) and nothing else, and
// code * s is exact in fp32. A power of two loses nothing against max|x| / 448 but at the
// subnormal end, since e4m3 is itself a floating type. A row holding an infinity or NaN
// gets the scale NaN and codes of zero: it reads back as NaN.
#pragma once

#include <cuda_fp8.h>

#include "kp_common.cuh"

namespace kpb {

// Error bit: a slot, page or position outside its table (kErrTimeout is 1, kErrSmemAlign 2).
constexpr unsigned kErrIndex = 4u;

constexpr int kMaxHeadDim = 256;

struct KvLayout {
  int64_t num_pages, page_size, heads, dim, page_stride;

  // First element of token `off` of page `page`, head `h`.
  __device__ __forceinline__ int64_t row(int64_t page, int64_t h, int64_t off) const {
    return page * page_stride + (h * page_size + off) * dim;
  }
  __device__ __forceinline__ int64_t scale(int64_t page, int64_t h, int64_t off) const {
    return (page * heads + h) * page_size + off;
  }
};

// log2 of n, -1 where n is no power of two.
inline int log2_of(int64_t n) {
  if ((n & (n - 1)) != 0) return -1;
  int log = 0;
  while (int64_t{1} << log < n) ++log;
  return log;
}

// Whether a note on a row's partials in paged_attention's workspace, (worker * 2 + slot of the
// first, how many), stays within the `workers` that there are. A note that no worker wrote
// (lengths that changed under the call) holds whatever the workspace held, so any pair of
// integers comes here; nothing is added that could pass 32 bits.
__host__ __device__ constexpr bool note_is_sound(int first_slot, int count, int workers) {
  return first_slot >= 0 && count >= 0 && first_slot >> 1 < workers &&
         count <= workers - (first_slot >> 1);
}

__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fffffff); }

// Scale of an e4m3 row whose largest magnitude has the bit pattern `amax` (sign cleared;
// patterns of infinities and NaNs are the largest, so an integer maximum carries them).
// `inv` is 1 / scale; 0 with the NaN scale, whose codes are zero.
__device__ __forceinline__ float e4m3_row_scale(uint32_t amax, float* inv) {
  if (amax >= 0x7f800000u) {
    *inv = 0.f;
    return nan_f();
  }
  if (amax == 0) {
    *inv = 1.f;
    return 1.f;
  }
  // 448 = 1.75 * 2^8: the exponent of amax - 8, one more where its fraction passes .75
  int e = static_cast<int>(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < 1 ? 1 : e;
  *inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}

// Code of x at 1/scale `inv` (exact product; rounds to nearest even). With inv = 0 (a row
// that is not finite) the code is 0, whatever x is.
__device__ __forceinline__ uint8_t e4m3_code(float x, float inv) {
  const float v = inv == 0.f ? 0.f : x * inv;
  return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float e4m3_value(uint8_t code) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}

// Element i of a row in a cache of type C (uint8_t: e4m3 codes, times the row's scale).
template <typename C>
__device__ __forceinline__ float cache_value(const C* row, int64_t i, float scale) {
  if constexpr (std::is_same_v<C, uint8_t>) {
    return e4m3_value(row[i]) * scale;
  } else {
    return to_f(row[i]);
  }
}

}  // namespace kpb
