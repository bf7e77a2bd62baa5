// RMS norm of every query and key head with the position rotation in the same pass
// (kp.qk_norm_rope), and its gradient (kp.qk_norm_rope_backward).
//
// A row is one head of one token, x in R^D. With r = 1 / sqrt(mean(x^2) + eps):
//   y = w * (x * r);   out = R(pos) y
// R turns the first `rot` elements in pairs (a, b) by the position's angles:
//   (a, b) -> (a cos - b sin, b cos + a sin)
// with the pair (i, i + rot/2), or (2i, 2i + 1) when interleaved; the rest passes through.
// cos_sin holds, per position, rot/2 cosines and then rot/2 sines in fp32.
// Backward, for g = d out:
//   dy = R(pos)^T g;  dw = sum over rows of dy * (x r);  dn = dy * w
//   dx = r * (dn - x r * mean(dn * x r))
// Everything is fp32 until the one rounding to the output type. A position outside the
// table gives NaN rows and sets kErrIndex.
//
//   variant 0  one warp per row, lanes strided over its elements
#include <algorithm>

#include "kp_kv_cache.cuh"

namespace kpb {
namespace {

constexpr int kWarpsPerCta = 8;
constexpr int kPerLane = kMaxHeadDim / kWarp;

struct RopeShape {
  int64_t tokens, q_heads, k_heads, dim, rot, max_pos;
  float eps;
  bool interleaved;
};

// The element that i rotates with, and whether i is the second of the pair.
__device__ __forceinline__ int partner(int i, int rot, bool interleaved, bool* second, int* angle) {
  const int half = rot / 2;
  if (interleaved) {
    *second = i & 1;
    *angle = i / 2;
    return i ^ 1;
  }
  *second = i >= half;
  *angle = *second ? i - half : i;
  return *second ? i - half : i + half;
}

// ------------------------------------------------------------------ variant 0

template <typename T>
__global__ void __launch_bounds__(kWarpsPerCta * kWarp)
rope_warp_row(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ wq,
              const T* __restrict__ wk, const float* __restrict__ cos_sin,
              const int64_t* __restrict__ positions, T* __restrict__ q_out,
              T* __restrict__ k_out, int64_t q_stride, int64_t k_stride, RopeShape sh,
              unsigned* err) {
  const int lane = threadIdx.x & (kWarp - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + threadIdx.x / kWarp;
  const int64_t heads = sh.q_heads + sh.k_heads;
  if (row >= sh.tokens * heads) return;
  const int64_t t = row / heads;
  const int64_t hh = row - t * heads;
  const bool is_q = hh < sh.q_heads;
  const int64_t h = is_q ? hh : hh - sh.q_heads;
  const int dim = static_cast<int>(sh.dim), rot = static_cast<int>(sh.rot);
  const T* x = is_q ? q + t * q_stride + h * dim : k + t * k_stride + h * dim;
  T* y = is_q ? q_out + (t * sh.q_heads + h) * dim : k_out + (t * sh.k_heads + h) * dim;
  const T* w = is_q ? wq : wk;

  float sq = 0.f;
  for (int i = lane; i < dim; i += kWarp) sq = fmaf(to_f(x[i]), to_f(x[i]), sq);
  float r = rsqrtf(warp_sum(sq) / static_cast<float>(dim) + sh.eps);
  int64_t pos = positions[t];
  if (pos < 0 || pos >= sh.max_pos) {
    if (lane == 0) atomicOr(err, kErrIndex);
    r = nan_f();
    pos = 0;
  }
  const float* cs = cos_sin + pos * rot;
  for (int i = lane; i < dim; i += kWarp) {
    float o = to_f(x[i]) * r * to_f(w[i]);
    if (i < rot && sh.max_pos > 0) {
      bool second;
      int a;
      const int j = partner(i, rot, sh.interleaved, &second, &a);
      const float other = to_f(x[j]) * r * to_f(w[j]);
      const float c = cs[a], s = cs[rot / 2 + a];
      o = second ? fmaf(o, c, other * s) : fmaf(o, c, -other * s);
    }
    y[i] = from_f<T>(o);
  }
}

// Rows of q then rows of k, strided over the grid's warps; each lane keeps the weight
// gradients of its elements, and a CTA writes its sums (in warp order) to
// partials[cta][2][dim].
template <typename T>
__global__ void __launch_bounds__(kWarpsPerCta * kWarp)
rope_back_warp_row(const T* __restrict__ gq, const T* __restrict__ gk, const T* __restrict__ q,
                   const T* __restrict__ k, const T* __restrict__ wq, const T* __restrict__ wk,
                   const float* __restrict__ cos_sin, const int64_t* __restrict__ positions,
                   T* __restrict__ dq, T* __restrict__ dk, float* __restrict__ partials,
                   int64_t gq_stride, int64_t gk_stride, int64_t q_stride, int64_t k_stride,
                   RopeShape sh, unsigned* err) {
  __shared__ float sums[kWarpsPerCta][kMaxHeadDim];
  const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
  const int dim = static_cast<int>(sh.dim), rot = static_cast<int>(sh.rot);
  for (int which = 0; which < 2; ++which) {
    const int64_t heads = which == 0 ? sh.q_heads : sh.k_heads;
    const T* w = which == 0 ? wq : wk;
    float acc[kPerLane] = {};
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + warp;
         row < sh.tokens * heads; row += static_cast<int64_t>(gridDim.x) * kWarpsPerCta) {
      const int64_t t = row / heads, h = row - t * heads;
      const T* x = (which == 0 ? q + t * q_stride : k + t * k_stride) + h * dim;
      const T* g = (which == 0 ? gq + t * gq_stride : gk + t * gk_stride) + h * dim;
      T* dx = (which == 0 ? dq : dk) + row * dim;
      int64_t pos = positions[t];
      const bool bad = pos < 0 || pos >= sh.max_pos;
      if (bad && lane == 0) atomicOr(err, kErrIndex);
      const float* cs = cos_sin + (bad ? 0 : pos) * rot;
      float sq = 0.f, inner = 0.f;
      float dy[kPerLane];
#pragma unroll
      for (int e = 0; e < kPerLane; ++e) {
        const int i = lane + e * kWarp;
        dy[e] = 0.f;
        if (i >= dim) continue;
        dy[e] = to_f(g[i]);
        if (i < rot && !bad) {
          bool second;
          int a;
          const int j = partner(i, rot, sh.interleaved, &second, &a);
          const float other = to_f(g[j]);
          const float c = cs[a], s = cs[rot / 2 + a];
          dy[e] = second ? fmaf(dy[e], c, -other * s) : fmaf(dy[e], c, other * s);
        }
        const float xi = to_f(x[i]);
        sq = fmaf(xi, xi, sq);
        inner = fmaf(dy[e] * to_f(w[i]), xi, inner);
      }
      const float inv_d = 1.f / static_cast<float>(dim);
      float r = rsqrtf(warp_sum(sq) * inv_d + sh.eps);
      if (bad) r = nan_f();
      const float m = warp_sum(inner) * inv_d * r;  // mean(dn * x r)
#pragma unroll
      for (int e = 0; e < kPerLane; ++e) {
        const int i = lane + e * kWarp;
        if (i >= dim) continue;
        const float xn = to_f(x[i]) * r;
        dx[i] = from_f<T>(r * fmaf(-xn, m, dy[e] * to_f(w[i])));
        acc[e] = fmaf(dy[e], xn, acc[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) sums[warp][lane + e * kWarp] = acc[e];
    __syncthreads();
    for (int i = threadIdx.x; i < dim; i += blockDim.x) {
      float total = 0.f;
      for (int j = 0; j < kWarpsPerCta; ++j) total += sums[j][i];
      partials[(static_cast<int64_t>(blockIdx.x) * 2 + which) * dim + i] = total;
    }
    __syncthreads();
  }
}

// dw[which][i] = sum over CTAs of partials[cta][which][i], in CTA order within each of the
// block's 8 rows of threads and then in row order: the same bits every time.
template <typename T>
__global__ void __launch_bounds__(256)
rope_weight_finish(const float* __restrict__ partials, int64_t ctas, int dim, T* dwq, T* dwk) {
  __shared__ float part[8][33];
  const int which = blockIdx.y;
  const int lane = threadIdx.x & (kWarp - 1), slice = threadIdx.x / kWarp;
  const int i = blockIdx.x * kWarp + lane;
  float s = 0.f;
  if (i < dim)
    for (int64_t c = slice; c < ctas; c += 8) s += partials[(c * 2 + which) * dim + i];
  part[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && i < dim) {
    s = 0.f;
    for (int j = 0; j < 8; ++j) s += part[j][lane];
    (which == 0 ? dwq : dwk)[i] = from_f<T>(s);
  }
}

// ------------------------------------------------------------------ launch

// CTAs of the backward's first kernel (each writes one partial of both weights).
int64_t back_ctas(const RopeShape& sh, int sms) {
  const int64_t rows = sh.tokens * std::max(sh.q_heads, sh.k_heads);
  return std::max<int64_t>(1, std::min<int64_t>(cdiv(rows, kWarpsPerCta), int64_t{4} * sms));
}

template <typename T>
int launch(const T* q, const T* k, const T* wq, const T* wk, const float* cos_sin,
           const int64_t* positions, T* q_out, T* k_out, int64_t q_stride, int64_t k_stride,
           const RopeShape& sh, unsigned* err, cudaStream_t s) {
  const int64_t rows = sh.tokens * (sh.q_heads + sh.k_heads);
  rope_warp_row<T><<<static_cast<unsigned>(cdiv(rows, kWarpsPerCta)), kWarpsPerCta * kWarp, 0, s>>>(
      q, k, wq, wk, cos_sin, positions, q_out, k_out, q_stride, k_stride, sh, err);
  KPB_LAUNCHED("qk_norm_rope");
  return KPB_OK;
}

template <typename T>
int launch_back(const T* gq, const T* gk, const T* q, const T* k, const T* wq, const T* wk,
                const float* cos_sin, const int64_t* positions, T* dq, T* dk, T* dwq, T* dwk,
                int64_t gq_stride, int64_t gk_stride, int64_t q_stride, int64_t k_stride,
                const RopeShape& sh, float* partials, unsigned* err, cudaStream_t s) {
  const int64_t ctas = back_ctas(sh, sm_count());
  rope_back_warp_row<T><<<static_cast<unsigned>(ctas), kWarpsPerCta * kWarp, 0, s>>>(
      gq, gk, q, k, wq, wk, cos_sin, positions, dq, dk, partials, gq_stride, gk_stride, q_stride,
      k_stride, sh, err);
  KPB_LAUNCHED("qk_norm_rope_backward");
  const dim3 grid(static_cast<unsigned>(cdiv(sh.dim, kWarp)), 2);
  rope_weight_finish<T><<<grid, 256, 0, s>>>(partials, ctas, static_cast<int>(sh.dim), dwq, dwk);
  KPB_LAUNCHED("qk_norm_rope_backward finish");
  return KPB_OK;
}

}  // namespace

size_t qk_norm_rope_backward_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t k_heads,
                                             int64_t dim) {
  RopeShape sh = {};
  sh.tokens = tokens;
  sh.q_heads = q_heads;
  sh.k_heads = k_heads;
  sh.dim = dim;
  // sized for the largest B200-class part, like the reduction's
  return static_cast<size_t>(back_ctas(sh, 256) * 2 * dim) * sizeof(float);
}

int qk_norm_rope(int variant, int dtype, const void* q, const void* k, const void* wq,
                 const void* wk, const float* cos_sin, const int64_t* positions, void* q_out,
                 void* k_out, int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t dim,
                 int64_t rot, int64_t max_pos, int64_t q_stride, int64_t k_stride, float eps,
                 bool interleaved, unsigned* err, cudaStream_t s) {
  const RopeShape sh{tokens, q_heads, k_heads, dim, rot, max_pos, eps, interleaved};
#define KPB_ROPE(T)                                                                       \
  launch<T>(static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(wq), \
            static_cast<const T*>(wk), cos_sin, positions, static_cast<T*>(q_out),        \
            static_cast<T*>(k_out), q_stride, k_stride, sh, err, s)
  switch (dtype) {
    case KPB_F32: return KPB_ROPE(float);
    case KPB_F16: return KPB_ROPE(__half);
    default: return KPB_ROPE(__nv_bfloat16);
  }
#undef KPB_ROPE
}

int qk_norm_rope_backward(int variant, int dtype, const void* gq, const void* gk, const void* q,
                          const void* k, const void* wq, const void* wk, const float* cos_sin,
                          const int64_t* positions, void* dq, void* dk, void* dwq, void* dwk,
                          int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t dim,
                          int64_t rot, int64_t max_pos, int64_t gq_stride, int64_t gk_stride,
                          int64_t q_stride, int64_t k_stride, float eps, bool interleaved,
                          void* ws, unsigned* err, cudaStream_t s) {
  const RopeShape sh{tokens, q_heads, k_heads, dim, rot, max_pos, eps, interleaved};
#define KPB_ROPE(T)                                                                            \
  launch_back<T>(static_cast<const T*>(gq), static_cast<const T*>(gk), static_cast<const T*>(q), \
                 static_cast<const T*>(k), static_cast<const T*>(wq), static_cast<const T*>(wk), \
                 cos_sin, positions, static_cast<T*>(dq), static_cast<T*>(dk),                 \
                 static_cast<T*>(dwq), static_cast<T*>(dwk), gq_stride, gk_stride, q_stride,   \
                 k_stride, sh, static_cast<float*>(ws), err, s)
  switch (dtype) {
    case KPB_F32: return KPB_ROPE(float);
    case KPB_F16: return KPB_ROPE(__half);
    default: return KPB_ROPE(__nv_bfloat16);
  }
#undef KPB_ROPE
}

}  // namespace kpb
