// Paged key/value cache: kp.kv_cache_write and kp.kv_cache_read.
//
// write: token t's Hkv key rows and value rows go to slot slots[t] = page * page_size +
// offset of their caches, as they are or as e4m3 codes with one scale per row (see
// kp_kv_cache.cuh). Slots below zero are padding and skipped.
// read: the same rows back out by slot, codes times scale; slots below zero give zeros.
//
//   variant 0  one warp per (token, head), lanes strided over the row's elements
//   variant 1  a row's 16-byte vectors (of the uncompressed side) over neighbouring lanes,
//              two to a lane; key and value row of a (token, head) loaded together before
//              either is used; one short-lived thread per four vectors, so the scheduler
//              keeps every SM's loads in flight. A row's largest magnitude is found on
//              packed 16-bit patterns. Bound by HBM, the e4m3 write nearly as much by its
//              instructions. Needs rows of whole vectors on vector boundaries; other layouts
//              take variant 0.
//
// Measured on B200 (6464 GB/s copy), 8 heads of 128, pages of 16: e4m3 write of 32768 bf16
// tokens 35 us (204 MB; 31.5 us at copy bandwidth), variant 0 125; bf16 read of 65536 tokens
// 83 us (537 MB; 83), variant 0 163; e4m3 read of 5001 tokens 6.2 us (31 MB; 4.8); plain bf16
// write of 32768 tokens 43.5 us (269 MB; 41.6). With one vector a lane and unpacked maxima the
// e4m3 write took 54 us, the reads 89 and 7.4.
#include "kp_kv_cache.cuh"

namespace kpb {
namespace {

constexpr int kWarpsPerCta = 8;

// (page, offset) of a slot. 0: in range, 1: padding (below zero), 2: out of range
// (recorded in *err). page_log: log2 of the page size, -1 where it is no power of two (a
// 64-bit division costs a fifth of the row's instructions).
__device__ __forceinline__ int locate(const KvLayout& lay, int page_log, int64_t slot,
                                      int64_t* page, int64_t* off, unsigned* err) {
  if (slot < 0) return 1;
  *page = page_log >= 0 ? slot >> page_log : slot / lay.page_size;
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
  if (locate(lay, -1, slots[t], &page, &off, err) != 0) return;
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
  const int state = locate(lay, -1, slots[t], &page, &off, err);
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

// ------------------------------------------------------------------ variant 1

constexpr int kVecThreads = 256;

// N codes of a vector, packed.
template <int N>
struct Codes {
  using type = std::conditional_t<N == 8, uint2, uint32_t>;
};

// The largest magnitude's bits of a vector: over packed pairs for the 16-bit types, whose
// patterns order as their fp32 values do (infinities and NaNs above the rest).
template <typename T>
__device__ __forceinline__ uint32_t max_bits(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu),
               max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
  } else {
    return __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                    __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
  }
}

// The pattern of max_bits over a row as that of an fp32 value.
template <typename T>
__device__ __forceinline__ uint32_t as_f32_bits(uint32_t v) {
  if constexpr (sizeof(T) == 4) {
    return v;
  } else {
    const uint32_t top = max(v & 0xffffu, v >> 16);
    if constexpr (std::is_same_v<T, __nv_bfloat16>) return top << 16;
    else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(top))));
  }
}

template <typename T>
__device__ __forceinline__ typename Codes<Vec<T>::kN>::type pack_codes(const float* f, float inv) {
  constexpr int N = Vec<T>::kN;
  uint32_t w[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    float g[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = f[4 * i + j] * inv;
    const uint32_t lo =
        __nv_cvt_float2_to_fp8x2(make_float2(g[0], g[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi =
        __nv_cvt_float2_to_fp8x2(make_float2(g[2], g[3]), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | hi << 16;
  }
  if constexpr (N == 8) return make_uint2(w[0], w[1]);
  else return w[0];
}

template <int N>
__device__ __forceinline__ void unpack_codes(const typename Codes<N>::type& v, float scale,
                                             float* f) {
  uint32_t w[2];
  if constexpr (N == 8) { w[0] = v.x; w[1] = v.y; } else { w[0] = v; }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const auto two = static_cast<__nv_fp8x2_storage_t>(w[i / 2] >> (i % 2 * 16));
    const float2 p = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
    f[2 * i] = p.x * scale;
    f[2 * i + 1] = p.y * scale;
  }
}

// 2^log_lanes lanes per row, V vectors each (lane, lane + lanes): lanes * V >= row vectors.
template <typename T, typename C, int V>
__global__ void __launch_bounds__(kVecThreads)
write_vector_rows(const T* __restrict__ k, const T* __restrict__ v,
                  const int64_t* __restrict__ slots, C* k_cache, C* v_cache, float* k_scale,
                  float* v_scale, int rows, int log_lanes, int page_log, int64_t k_stride,
                  int64_t v_stride, KvLayout lay, unsigned* err) {
  constexpr int N = Vec<T>::kN;
  const int lanes = 1 << log_lanes, lane = threadIdx.x & (lanes - 1);
  const int64_t group = (static_cast<int64_t>(blockIdx.x) * kVecThreads + threadIdx.x) >> log_lanes;
  const bool live = group < rows;  // a group past the last row still joins the shuffles
  const int row = static_cast<int>(group);
  const int heads = static_cast<int>(lay.heads), nv = static_cast<int>(lay.dim) / N;
  const int t = live ? row / heads : 0, h = live ? row - t * heads : 0;
  const uint64_t pol = evict_first_policy();
  const uint4* src[2] = {reinterpret_cast<const uint4*>(k + t * k_stride + h * lay.dim),
                         reinterpret_cast<const uint4*>(v + t * v_stride + h * lay.dim)};
  uint4 raw[2][V];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int j = lane + i * lanes;
      raw[w][i] = live && j < nv ? ld_stream(src[w] + j, pol) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  int64_t page = 0, off = 0;
  const bool store = live && locate(lay, page_log, slots[t], &page, &off, err) == 0;
  const int64_t at = lay.row(page, h, off);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    C* y = (w == 0 ? k_cache : v_cache) + at;
    if constexpr (std::is_same_v<C, uint8_t>) {
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t top = max_bits<T>(raw[w][i]);
        amax = sizeof(T) == 4 ? max(amax, top) : __vmaxu2(amax, top);
      }
      for (int o = lanes >> 1; o > 0; o >>= 1) {
        const uint32_t other = __shfl_xor_sync(kFull, amax, o);
        amax = sizeof(T) == 4 ? max(amax, other) : __vmaxu2(amax, other);
      }
      float inv;
      const float s = e4m3_row_scale(as_f32_bits<T>(amax), &inv);
      if (!store) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = lane + i * lanes;
        float f[N];
        unpack<T>(raw[w][i], f);
        typename Codes<N>::type codes = pack_codes<T>(f, inv);
        // a row that is not finite: its NaN * 0 would be no code of 0
        if (inv == 0.f) codes = typename Codes<N>::type{};
        if (j < nv) reinterpret_cast<typename Codes<N>::type*>(y)[j] = codes;
      }
      if (lane == 0) (w == 0 ? k_scale : v_scale)[lay.scale(page, h, off)] = s;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = lane + i * lanes;
        if (store && j < nv) reinterpret_cast<uint4*>(y)[j] = raw[w][i];
      }
    }
  }
}

template <typename T, typename C, int V>
__global__ void __launch_bounds__(kVecThreads)
read_vector_rows(const C* __restrict__ k_cache, const C* __restrict__ v_cache,
                 const int64_t* __restrict__ slots, const float* __restrict__ k_scale,
                 const float* __restrict__ v_scale, T* __restrict__ k, T* __restrict__ v,
                 int rows, int log_lanes, int page_log, KvLayout lay, unsigned* err) {
  constexpr int N = Vec<T>::kN;
  using Held = std::conditional_t<std::is_same_v<C, uint8_t>, typename Codes<N>::type, uint4>;
  const int lanes = 1 << log_lanes, lane = threadIdx.x & (lanes - 1);
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kVecThreads + threadIdx.x) >> log_lanes;
  if (row >= rows) return;
  const int heads = static_cast<int>(lay.heads), nv = static_cast<int>(lay.dim) / N;
  const int t = static_cast<int>(row) / heads, h = static_cast<int>(row) - t * heads;
  int64_t page = 0, off = 0;
  const int state = locate(lay, page_log, slots[t], &page, &off, err);
  const int64_t at = lay.row(page, h, off);
  Held raw[2][V] = {};
  float scale[2] = {1.f, 1.f};
  if (state == 0) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const Held* src = reinterpret_cast<const Held*>((w == 0 ? k_cache : v_cache) + at);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = lane + i * lanes;
        if (j < nv) raw[w][i] = __ldg(src + j);
      }
    }
    if constexpr (std::is_same_v<C, uint8_t>) {
      scale[0] = k_scale[lay.scale(page, h, off)];
      scale[1] = v_scale[lay.scale(page, h, off)];
    }
  }
  const float fill = state == 1 ? 0.f : nan_f();  // padding, or a slot out of range
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint4* y = reinterpret_cast<uint4*>((w == 0 ? k : v) + row * lay.dim);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int j = lane + i * lanes;
      if (j >= nv) continue;
      if constexpr (std::is_same_v<C, T>) {
        if (state == 0) {
          st_stream(y + j, raw[w][i]);
          continue;
        }
      }
      float f[N];
      if constexpr (std::is_same_v<C, uint8_t>) unpack_codes<N>(raw[w][i], scale[w], f);
      if (state != 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = fill;
      }
      st_stream(y + j, pack<T>(f));
    }
  }
}

// ------------------------------------------------------------------ launch

uintptr_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Rows of the cache in whole vectors of N elements on their boundaries, N being 16 bytes of
// T; the scratch of lanes per row and vectors per lane.
template <typename T, typename C>
bool vector_rows(const KvLayout& lay, const void* k_cache, const void* v_cache) {
  constexpr int N = Vec<T>::kN;
  return lay.dim % N == 0 && (addr(k_cache) | addr(v_cache)) % (N * sizeof(C)) == 0 &&
         (lay.num_pages < 2 || lay.page_stride % N == 0);
}

// Two vectors of each row to a lane, so that a row's fixed work (its slot, its scale) falls
// on half the threads; 32 lanes then hold the longest row (fp32, D = 256).
constexpr int kPerRowLane = 2;

int lanes_log2(int64_t vectors) {
  int log = 0;
  while ((kPerRowLane << log) < vectors) ++log;
  return log;
}

template <typename T, typename C>
int launch_write(int variant, const void* k, const void* v, const int64_t* slots, void* k_cache,
                 void* v_cache, float* k_scale, float* v_scale, int64_t tokens, int64_t k_stride,
                 int64_t v_stride, const KvLayout& lay, unsigned* err, cudaStream_t s) {
  constexpr int N = Vec<T>::kN;
  if (variant == 1 && vector_rows<T, C>(lay, k_cache, v_cache) &&
      (addr(k) | addr(v)) % 16 == 0 && (tokens < 2 || (k_stride | v_stride) % N == 0)) {
    const int64_t nv = lay.dim / N;
    const int log = lanes_log2(nv), rows = static_cast<int>(tokens * lay.heads);
    const auto ctas = static_cast<unsigned>(cdiv(static_cast<int64_t>(rows) << log, kVecThreads));
    write_vector_rows<T, C, kPerRowLane><<<ctas, kVecThreads, 0, s>>>(
        static_cast<const T*>(k), static_cast<const T*>(v), slots, static_cast<C*>(k_cache),
        static_cast<C*>(v_cache), k_scale, v_scale, rows, log, log2_of(lay.page_size), k_stride,
        v_stride, lay, err);
    KPB_LAUNCHED("kv_cache_write vector rows");
    return KPB_OK;
  }
  const auto ctas = static_cast<unsigned>(cdiv(tokens * lay.heads, kWarpsPerCta));
  write_warp_row<T, C><<<ctas, kWarpsPerCta * kWarp, 0, s>>>(
      static_cast<const T*>(k), static_cast<const T*>(v), slots, static_cast<C*>(k_cache),
      static_cast<C*>(v_cache), k_scale, v_scale, tokens, k_stride, v_stride, lay, err);
  KPB_LAUNCHED("kv_cache_write");
  return KPB_OK;
}

template <typename T, typename C>
int launch_read(int variant, const void* k_cache, const void* v_cache, const int64_t* slots,
                const float* k_scale, const float* v_scale, void* k, void* v, int64_t tokens,
                const KvLayout& lay, unsigned* err, cudaStream_t s) {
  constexpr int N = Vec<T>::kN;
  if (variant == 1 && vector_rows<T, C>(lay, k_cache, v_cache) && (addr(k) | addr(v)) % 16 == 0) {
    const int64_t nv = lay.dim / N;
    const int log = lanes_log2(nv), rows = static_cast<int>(tokens * lay.heads);
    const auto ctas = static_cast<unsigned>(cdiv(static_cast<int64_t>(rows) << log, kVecThreads));
    read_vector_rows<T, C, kPerRowLane><<<ctas, kVecThreads, 0, s>>>(
        static_cast<const C*>(k_cache), static_cast<const C*>(v_cache), slots, k_scale, v_scale,
        static_cast<T*>(k), static_cast<T*>(v), rows, log, log2_of(lay.page_size), lay,
        err);
    KPB_LAUNCHED("kv_cache_read vector rows");
    return KPB_OK;
  }
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
#define KPB_WRITE(T, C)                                                                  \
  launch_write<T, C>(variant, k, v, slots, k_cache, v_cache, k_scale, v_scale, tokens,   \
                     k_stride, v_stride, lay, err, s)
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
  launch_read<T, C>(variant, k_cache, v_cache, slots, k_scale, v_scale, k, v, tokens, lay, err, s)
  const bool q = cache_dtype == KPB_E4M3;
  switch (dtype) {
    case KPB_F32: return q ? KPB_READ(float, uint8_t) : KPB_READ(float, float);
    case KPB_F16: return q ? KPB_READ(__half, uint8_t) : KPB_READ(__half, __half);
    default: return q ? KPB_READ(__nv_bfloat16, uint8_t) : KPB_READ(__nv_bfloat16, __nv_bfloat16);
  }
#undef KPB_READ
}

}  // namespace kpb
