// Paged key/value cache: kp.kv_cache_write and kp.kv_cache_read.
//
// write: token t's Hkv key rows and value rows go to slot slots[t] = page * page_size +
// offset of their caches, as they are or as e4m3 codes with one scale per row (see
// kp_kv_cache.cuh). Slots below zero are padding and skipped.
// read: the same rows back out by slot, codes times scale; slots below zero give zeros.
//
//   variant 0  one warp per (token, head), lanes strided over the row's elements
#include "kp_kv_cache.cuh"

namespace kpb {
namespace {

constexpr int kWarpsPerCta = 8;

// (page, offset) of a slot. 0: in range, 1: padding (below zero), 2: out of range
// (recorded in *err).
__device__ __forceinline__ int locate(const KvLayout& lay, int64_t slot, int64_t* page,
                                      int64_t* off, unsigned* err) {
  if (slot < 0) return 1;
  *page = slot / lay.page_size;
  *off = slot - *page * lay.page_size;
  if (*page >= lay.num_pages) {
    atomicOr(err, kErrIndex);
    return 2;
  }
  return 0;
}

// ------------------------------------------------------------------ variant 0

template <typename T, typename C>
__global__ void __launch_bounds__(kWarpsPerCta * kWarp)
write_warp_row(const T* __restrict__ k, const T* __restrict__ v,
               const int64_t* __restrict__ slots, C* k_cache, C* v_cache, float* k_scale,
               float* v_scale, int64_t tokens, int64_t k_stride, int64_t v_stride, KvLayout lay,
               unsigned* err) {
  const int lane = threadIdx.x & (kWarp - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + threadIdx.x / kWarp;
  if (row >= tokens * lay.heads) return;
  const int64_t t = row / lay.heads, h = row - t * lay.heads;
  int64_t page, off;
  if (locate(lay, slots[t], &page, &off, err) != 0) return;
  const int64_t at = lay.row(page, h, off), sat = lay.scale(page, h, off);
  for (int which = 0; which < 2; ++which) {
    const T* x = which == 0 ? k + t * k_stride + h * lay.dim : v + t * v_stride + h * lay.dim;
    C* y = (which == 0 ? k_cache : v_cache) + at;
    if constexpr (std::is_same_v<C, uint8_t>) {
      uint32_t amax = 0;
      for (int64_t i = lane; i < lay.dim; i += kWarp)
        amax = max(amax, __float_as_uint(to_f(x[i])) & 0x7fffffffu);
      amax = __reduce_max_sync(kFull, amax);
      float inv;
      const float s = e4m3_row_scale(amax, &inv);
      for (int64_t i = lane; i < lay.dim; i += kWarp) y[i] = e4m3_code(to_f(x[i]), inv);
      if (lane == 0) (which == 0 ? k_scale : v_scale)[sat] = s;
    } else {
      for (int64_t i = lane; i < lay.dim; i += kWarp) y[i] = x[i];
    }
  }
}

template <typename T, typename C>
__global__ void __launch_bounds__(kWarpsPerCta * kWarp)
read_warp_row(const C* __restrict__ k_cache, const C* __restrict__ v_cache,
              const int64_t* __restrict__ slots, const float* __restrict__ k_scale,
              const float* __restrict__ v_scale, T* __restrict__ k, T* __restrict__ v,
              int64_t tokens, KvLayout lay, unsigned* err) {
  const int lane = threadIdx.x & (kWarp - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + threadIdx.x / kWarp;
  if (row >= tokens * lay.heads) return;
  const int64_t t = row / lay.heads, h = row - t * lay.heads;
  int64_t page = 0, off = 0;
  const int state = locate(lay, slots[t], &page, &off, err);
  const int64_t at = lay.row(page, h, off), sat = lay.scale(page, h, off);
  for (int which = 0; which < 2; ++which) {
    T* y = (which == 0 ? k : v) + row * lay.dim;
    if (state != 0) {  // padding reads as zeros, a slot out of range as NaN
      for (int64_t i = lane; i < lay.dim; i += kWarp) y[i] = from_f<T>(state == 1 ? 0.f : nan_f());
      continue;
    }
    const C* x = (which == 0 ? k_cache : v_cache) + at;
    if constexpr (std::is_same_v<C, T>) {
      for (int64_t i = lane; i < lay.dim; i += kWarp) y[i] = x[i];
    } else {
      const float s = (which == 0 ? k_scale : v_scale)[sat];
      for (int64_t i = lane; i < lay.dim; i += kWarp) y[i] = from_f<T>(cache_value(x, i, s));
    }
  }
}

// ------------------------------------------------------------------ launch

template <typename T, typename C>
int launch_write(const void* k, const void* v, const int64_t* slots, void* k_cache,
                 void* v_cache, float* k_scale, float* v_scale, int64_t tokens, int64_t k_stride,
                 int64_t v_stride, const KvLayout& lay, unsigned* err, cudaStream_t s) {
  const auto ctas = static_cast<unsigned>(cdiv(tokens * lay.heads, kWarpsPerCta));
  write_warp_row<T, C><<<ctas, kWarpsPerCta * kWarp, 0, s>>>(
      static_cast<const T*>(k), static_cast<const T*>(v), slots, static_cast<C*>(k_cache),
      static_cast<C*>(v_cache), k_scale, v_scale, tokens, k_stride, v_stride, lay, err);
  KPB_LAUNCHED("kv_cache_write");
  return KPB_OK;
}

template <typename T, typename C>
int launch_read(const void* k_cache, const void* v_cache, const int64_t* slots,
                const float* k_scale, const float* v_scale, void* k, void* v, int64_t tokens,
                const KvLayout& lay, unsigned* err, cudaStream_t s) {
  const auto ctas = static_cast<unsigned>(cdiv(tokens * lay.heads, kWarpsPerCta));
  read_warp_row<T, C><<<ctas, kWarpsPerCta * kWarp, 0, s>>>(
      static_cast<const C*>(k_cache), static_cast<const C*>(v_cache), slots, k_scale, v_scale,
      static_cast<T*>(k), static_cast<T*>(v), tokens, lay, err);
  KPB_LAUNCHED("kv_cache_read");
  return KPB_OK;
}

}  // namespace

int kv_cache_write(int variant, int dtype, int cache_dtype, const void* k, const void* v,
                   const int64_t* slots, void* k_cache, void* v_cache, float* k_scale,
                   float* v_scale, int64_t tokens, int64_t k_stride, int64_t v_stride,
                   const KvLayout& lay, unsigned* err, cudaStream_t s) {
#define KPB_WRITE(T, C)                                                                      \
  launch_write<T, C>(k, v, slots, k_cache, v_cache, k_scale, v_scale, tokens, k_stride,      \
                     v_stride, lay, err, s)
  const bool q = cache_dtype == KPB_E4M3;
  switch (dtype) {
    case KPB_F32: return q ? KPB_WRITE(float, uint8_t) : KPB_WRITE(float, float);
    case KPB_F16: return q ? KPB_WRITE(__half, uint8_t) : KPB_WRITE(__half, __half);
    default: return q ? KPB_WRITE(__nv_bfloat16, uint8_t) : KPB_WRITE(__nv_bfloat16, __nv_bfloat16);
  }
#undef KPB_WRITE
}

int kv_cache_read(int variant, int dtype, int cache_dtype, const void* k_cache,
                  const void* v_cache, const int64_t* slots, const float* k_scale,
                  const float* v_scale, void* k, void* v, int64_t tokens, const KvLayout& lay,
                  unsigned* err, cudaStream_t s) {
#define KPB_READ(T, C) \
  launch_read<T, C>(k_cache, v_cache, slots, k_scale, v_scale, k, v, tokens, lay, err, s)
  const bool q = cache_dtype == KPB_E4M3;
  switch (dtype) {
    case KPB_F32: return q ? KPB_READ(float, uint8_t) : KPB_READ(float, float);
    case KPB_F16: return q ? KPB_READ(__half, uint8_t) : KPB_READ(__half, __half);
    default: return q ? KPB_READ(__nv_bfloat16, uint8_t) : KPB_READ(__nv_bfloat16, __nv_bfloat16);
  }
#undef KPB_READ
}

}  // namespace kpb
