// Attention of one new token per sequence over the paged cache (kp.paged_attention):
//   o[b, h] = softmax_j(scale * q[b, h] . K[j]) V[j],   j < seq_lens[b],
// K[j], V[j] the rows of key head h / (Hq / Hkv) in page block_table[b][j / page_size] at
// offset j % page_size. The softmax's maximum, sum and the weighted sum of values are
// fp32, carried along the keys in one pass. A sequence of length 0 gives zeros. Nothing
// past a sequence's last key is read. A page outside the cache gives that sequence's heads
// NaN and sets kErrIndex; a length past the table's width is cut to it and sets kErrIndex.
//
//   variant 0  one CTA per (sequence, query head): four warps take every fourth key each,
//              lanes strided over the row's elements, and join at the end
#include "kp_kv_cache.cuh"

namespace kpb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPerLane = kMaxHeadDim / kWarp;

struct PagedShape {
  int64_t batch, q_heads, max_pages, q_stride, table_stride;
  float scale;
  KvLayout lay;
};

// Keys of sequence b: its length, cut to what the table can hold.
__device__ __forceinline__ int64_t keys_of(const int* __restrict__ seq_lens, int64_t b,
                                           const PagedShape& sh, unsigned* err) {
  int64_t n = seq_lens[b];
  const int64_t most = sh.max_pages * sh.lay.page_size;
  if (n > most || n < 0) {
    atomicOr(err, kErrIndex);
    n = n < 0 ? 0 : most;
  }
  return n;
}

// ------------------------------------------------------------------ variant 0

template <typename T, typename C>
__global__ void __launch_bounds__(128)
paged_cta_head(const T* __restrict__ q, const C* __restrict__ k_cache,
               const C* __restrict__ v_cache, const int* __restrict__ table,
               const int* __restrict__ seq_lens, const float* __restrict__ k_scale,
               const float* __restrict__ v_scale, T* __restrict__ o, PagedShape sh,
               unsigned* err) {
  __shared__ float s_m[4], s_l[4], s_o[4][kMaxHeadDim];
  const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
  const int64_t b = blockIdx.x / sh.q_heads, h = blockIdx.x - b * sh.q_heads;
  const int64_t hk = h / (sh.q_heads / sh.lay.heads);
  const int dim = static_cast<int>(sh.lay.dim);
  const int64_t n = keys_of(seq_lens, b, sh, err);
  T* out = o + (b * sh.q_heads + h) * dim;
  float qr[kPerLane], acc[kPerLane] = {};
#pragma unroll
  for (int e = 0; e < kPerLane; ++e) {
    const int i = lane + e * kWarp;
    qr[e] = i < dim ? to_f(q[b * sh.q_stride + h * dim + i]) * (sh.scale * kLog2e) : 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = warp; j < n; j += 4) {
    const int64_t page = table[b * sh.table_stride + j / sh.lay.page_size];
    if (page < 0 || page >= sh.lay.num_pages) {
      if (lane == 0) atomicOr(err, kErrIndex);
      l = nan_f();
      continue;
    }
    const int64_t off = j % sh.lay.page_size;
    const int64_t at = sh.lay.row(page, hk, off);
    float ks = 1.f, vs = 1.f;
    if constexpr (std::is_same_v<C, uint8_t>) {
      ks = k_scale[sh.lay.scale(page, hk, off)];
      vs = v_scale[sh.lay.scale(page, hk, off)];
    }
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) {
      const int i = lane + e * kWarp;
      if (i < dim) dot = fmaf(qr[e], cache_value(k_cache + at, i, ks), dot);
    }
    const float s = warp_sum(dot);
    const float m_new = fmaxf(m, s);  // a NaN score stays out of the maximum: its weight is NaN
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - base), p = exp2f(s - base);
    l = fmaf(l, alpha, p);
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) {
      const int i = lane + e * kWarp;
      if (i < dim) acc[e] = fmaf(acc[e], alpha, p * cache_value(v_cache + at, i, vs));
    }
    m = m_new;
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < kPerLane; ++e) s_o[warp][lane + e * kWarp] = acc[e];
  __syncthreads();
  float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  if (top == -INFINITY) top = 0.f;
  float sum = 0.f, f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = exp2f(s_m[i] - top);
    sum = fmaf(s_l[i], f[i], sum);
  }
  for (int i = threadIdx.x; i < dim; i += blockDim.x) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v = fmaf(s_o[w][i], f[w], v);
    out[i] = from_f<T>(n == 0 ? 0.f : v / sum);
  }
}

// ------------------------------------------------------------------ launch

template <typename T, typename C>
int launch(const void* q, const void* k_cache, const void* v_cache, const int* table,
           const int* seq_lens, const float* k_scale, const float* v_scale, void* o,
           const PagedShape& sh, unsigned* err, cudaStream_t s) {
  paged_cta_head<T, C><<<static_cast<unsigned>(sh.batch * sh.q_heads), 128, 0, s>>>(
      static_cast<const T*>(q), static_cast<const C*>(k_cache), static_cast<const C*>(v_cache),
      table, seq_lens, k_scale, v_scale, static_cast<T*>(o), sh, err);
  KPB_LAUNCHED("paged_attention variant 0");
  return KPB_OK;
}

}  // namespace

size_t paged_attention_workspace_bytes(int variant, int64_t batch, int64_t q_heads,
                                       int64_t k_heads, int64_t dim, int64_t max_len) {
  return 0;
}

int paged_attention(int variant, int dtype, int cache_dtype, const void* q, const void* k_cache,
                    const void* v_cache, const int* table, const int* seq_lens,
                    const float* k_scale, const float* v_scale, void* o, int64_t batch,
                    int64_t q_heads, int64_t max_pages, int64_t q_stride, int64_t table_stride,
                    float scale, const KvLayout& lay, void* ws, size_t ws_bytes, unsigned* err,
                    cudaStream_t s) {
  const PagedShape sh{batch, q_heads, max_pages, q_stride, table_stride, scale, lay};
#define KPB_PAGED(T, C) \
  launch<T, C>(q, k_cache, v_cache, table, seq_lens, k_scale, v_scale, o, sh, err, s)
  const bool e4m3 = cache_dtype == KPB_E4M3;
  switch (dtype) {
    case KPB_F32: return e4m3 ? KPB_PAGED(float, uint8_t) : KPB_PAGED(float, float);
    case KPB_F16: return e4m3 ? KPB_PAGED(__half, uint8_t) : KPB_PAGED(__half, __half);
    default:
      return e4m3 ? KPB_PAGED(__nv_bfloat16, uint8_t) : KPB_PAGED(__nv_bfloat16, __nv_bfloat16);
  }
#undef KPB_PAGED
}

}  // namespace kpb
