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
//   variant 1  a lane holds two vectors of a row that rotate with one another (i and
//              i + rot/2), so no value crosses lanes but the row's sums; rows of D = 128
//              16-bit values take 8 lanes. The angles and weights of a token are read (and
//              multiplied) once for several heads, and the arithmetic is on packed fp32
//              pairs: with the bytes of a row in registers or in a shared-memory ring, what
//              bounds both kernels is the instructions and the latency between a token's
//              position and its angles. The backward is one wave of CTAs, some for q and
//              some for k, each lane adding its elements' weight gradients in registers over
//              all its rows; a second small kernel adds the CTAs' sums in a fixed order.
//              Needs both parts of the row (rotated and not) in whole pairs of vectors on
//              vector boundaries (16 bytes, or 8 for 16-bit types); other layouts take
//              variant 0.
//
// Measured on B200 (6464 GB/s copy), 16384 tokens, 32 + 8 heads of 128, bf16: forward 59 us
// (344 MB; 53 us at copy bandwidth), variant 0 265; backward 95 us (512 MB; 79), variant 0
// 955. 64 tokens: forward 2.9 us. Other shapes are further off, variant 1's turns and lanes
// being padded: heads of 80 and 96 elements take 8 lanes for 5 and 6 pairs (32768 tokens, 24 + 8
// heads: 86 us for 54 at copy bandwidth, 88 for 64), and a turn costs four heads where it has
// one (4 + 1 heads of 128: 26 us for 16).
#include <algorithm>

#include "kp_kv_cache.cuh"
#include "kp_sm100.cuh"

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

// ------------------------------------------------------------------ variant 1

constexpr int kRopeThreads = 128;  // forward
constexpr int kVecThreads = 256;   // backward

template <int Bytes>
struct Raw {
  using type = std::conditional_t<Bytes == 16, uint4, uint2>;
};

template <typename T, int VE>
using RawOf = typename Raw<VE * static_cast<int>(sizeof(T))>::type;

// Streamed load of one vector: not kept in L1, first to leave L2.
template <typename R>
__device__ __forceinline__ R load_stream(const void* p, uint64_t pol) {
  if constexpr (sizeof(R) == 16) {
    return ld_stream(p, pol);
  } else {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::cache_hint.v2.u32 {%0,%1}, [%2], %3;"
                 : "=r"(v.x), "=r"(v.y) : "l"(p), "l"(pol));
    return v;
  }
}

// A vector's VE elements as VE / 2 packed pairs of floats, and back.
template <typename T, int VE, typename R>
__device__ __forceinline__ void unpack_raw(const R& v, float2* f) {
  float g[8];
  if constexpr (sizeof(R) == 16) {
    unpack<T>(v, g);
  } else {
    unpack<T>(make_uint4(v.x, v.y, 0u, 0u), g);
  }
#pragma unroll
  for (int e = 0; e < VE / 2; ++e) f[e] = make_float2(g[2 * e], g[2 * e + 1]);
}

template <typename T, int VE>
__device__ __forceinline__ void store_raw(T* p, const float2* f) {
  float g[8] = {};
#pragma unroll
  for (int e = 0; e < VE / 2; ++e) {
    g[2 * e] = f[e].x;
    g[2 * e + 1] = f[e].y;
  }
  const uint4 v = pack<T>(g);
  if constexpr (VE * sizeof(T) == 16) {
    st_stream(p, v);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(v.x, v.y);
  }
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 neg2(float2 v) { return make_float2(-v.x, -v.y); }

// Where pair `p` of a row lies: vectors at a and b, turned by the angles from `angle` on
// (vector a) and `angle2` on (vector b; adjacent pairs only).
struct PairPlace {
  int a, b, angle, angle2;
  bool turned;
};

template <int VE, bool kAdjacent>
__device__ __forceinline__ PairPlace pair_place(int p, const RopeShape& sh) {
  const int rot = static_cast<int>(sh.rot), dim = static_cast<int>(sh.dim);
  PairPlace w;
  w.turned = p * 2 * VE < rot;
  const int from = w.turned ? 0 : rot, half = (w.turned ? rot : dim - rot) / 2;
  w.a = from + (p * VE - (w.turned ? 0 : rot / 2));
  w.b = w.a + half;
  w.angle = kAdjacent ? w.a / 2 : w.a;
  w.angle2 = w.b / 2;
  return w;
}

// Cosines and sines for the lane's two vectors, as packed pairs. Pairs rot/2 apart share
// them: (a, b) turns to (a c - b s, b c + a s), and cb, sb are left alone. With adjacent
// pairs a turns to a * ca + swapped(a) * sa, sa = (-sin, sin), and b likewise.
template <int VE, bool kAdjacent>
__device__ __forceinline__ void load_angles(const float* __restrict__ row, const PairPlace& w,
                                            const RopeShape& sh, bool ok, float2* ca, float2* sa,
                                            float2* cb, float2* sb) {
  const int half = static_cast<int>(sh.rot) / 2;
#pragma unroll
  for (int e = 0; e < VE / 2; ++e) {
    ca[e] = both(1.f);
    sa[e] = both(0.f);
    if constexpr (kAdjacent) {
      cb[e] = both(1.f);
      sb[e] = both(0.f);
    }
  }
  if (!w.turned || !ok) return;
  if constexpr (!kAdjacent) {
#pragma unroll
    for (int e = 0; e < VE; e += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(row + w.angle + e));
      const float4 y = __ldg(reinterpret_cast<const float4*>(row + half + w.angle + e));
      ca[e / 2] = make_float2(x.x, x.y);
      ca[e / 2 + 1] = make_float2(x.z, x.w);
      sa[e / 2] = make_float2(y.x, y.y);
      sa[e / 2 + 1] = make_float2(y.z, y.w);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE / 2; ++e) {
      ca[e] = both(__ldg(row + w.angle + e));
      cb[e] = both(__ldg(row + w.angle2 + e));
      const float s = __ldg(row + half + w.angle + e), s2 = __ldg(row + half + w.angle2 + e);
      sa[e] = make_float2(-s, s);
      sb[e] = make_float2(-s2, s2);
    }
  }
}

__device__ __forceinline__ float2 swapped(float2 v) { return make_float2(v.y, v.x); }

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

__device__ __forceinline__ float2 group_sum2(float2 v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(kFull, v.x, o);
    v.y += __shfl_xor_sync(kFull, v.y, o);
  }
  return v;
}

// A turn of a group of 2^log_lanes lanes is HPG heads (all of q or all of k) of one token.
// kRing: one wave of CTAs, a group's turns `step` apart, each thread's own vectors through
// its own slots of a shared-memory ring (cp.async, kForwardStages - 1 turns ahead). Else one
// turn to a group, its vectors read into registers.
constexpr int kForwardStages = 2;  // `stage ^ 1` below is the other one

template <typename T, int VE, int HPG, bool kAdjacent, bool kRing>
__global__ void __launch_bounds__(kRopeThreads, kRing ? 5 : 4)
rope_vector_pairs(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ wq,
                  const T* __restrict__ wk, const float* __restrict__ cos_sin,
                  const int64_t* __restrict__ positions, T* __restrict__ q_out,
                  T* __restrict__ k_out, int64_t q_stride, int64_t k_stride, int log_lanes,
                  RopeShape sh, unsigned* err) {
  using R = RawOf<T, VE>;
  extern __shared__ __align__(16) unsigned char ring[];  // [stage][head][a, b][thread]
  const int lanes = 1 << log_lanes, lane = threadIdx.x & (lanes - 1);
  const int hq = static_cast<int>(sh.q_heads), hk = static_cast<int>(sh.k_heads);
  const int dim = static_cast<int>(sh.dim);
  const uint32_t q_parts = (hq + HPG - 1) / HPG, parts = q_parts + (hk + HPG - 1) / HPG;
  const int64_t items = sh.tokens * parts;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kRopeThreads) >> log_lanes;
  const int64_t step = (static_cast<int64_t>(gridDim.x) * kRopeThreads) >> log_lanes;
  const int in_cta = static_cast<int>(threadIdx.x) >> log_lanes;
  const PairPlace pl = pair_place<VE, kAdjacent>(lane, sh);
  const bool holds = lane * 2 * VE < dim;
  const uint64_t pol = evict_first_policy();

  struct Turn {
    uint32_t t;
    int h0, heads, mine;
    bool is_q, live;
  };
  const auto turn_of = [&](int64_t item) {
    Turn n;
    n.live = item < items;  // the rest still join the shuffles
    n.t = n.live ? static_cast<uint32_t>(item) / parts : 0;
    const uint32_t part = n.live ? static_cast<uint32_t>(item) - n.t * parts : 0;
    n.is_q = part < q_parts;
    n.h0 = static_cast<int>(n.is_q ? part : part - q_parts) * HPG;
    n.heads = n.is_q ? hq : hk;
    n.mine = n.live && holds ? min(HPG, n.heads - n.h0) : 0;
    return n;
  };
  const auto row_of = [&](const Turn& n) {
    return (n.is_q ? q + n.t * q_stride : k + n.t * k_stride) + static_cast<int64_t>(n.h0) * dim;
  };
  const auto slot = [&](int stage, int i, int v) {
    return ((stage * HPG + i) * 2 + v) * kRopeThreads + static_cast<int>(threadIdx.x);
  };
  int64_t ahead = first + in_cta, next_pos = 0;
  const auto load = [&](int stage) {
    const Turn n = turn_of(ahead);
    const T* x = row_of(n);
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      if (i >= n.mine) break;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const uint32_t dst = smem_u32(ring) + slot(stage, i, v) * static_cast<uint32_t>(sizeof(R));
        const T* src = x + i * dim + (v == 0 ? pl.a : pl.b);
        if constexpr (sizeof(R) == 16) cp_async16(dst, src);
        else cp_async8(dst, src, true);
      }
    }
    cp_async_commit();
    next_pos = n.live ? positions[n.t] : 0;
    ahead += step;
  };
  int stage = 0;
  if constexpr (kRing) load(0);

  // every lane of the CTA takes the same number of turns: the shuffles need whole warps
  for (int64_t base = first; base < items; base += step) {
    const Turn n = turn_of(base + in_cta);
    R raw[HPG][2];
    int64_t pos;
    if constexpr (kRing) {
      pos = next_pos;
      load(stage ^ 1);
    } else {
      const T* x = row_of(n);
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        raw[i][0] = raw[i][1] = R{};
        if (i < n.mine) {
          raw[i][0] = load_stream<R>(x + i * dim + pl.a, pol);
          raw[i][1] = load_stream<R>(x + i * dim + pl.b, pol);
        }
      }
      pos = n.live ? positions[n.t] : 0;
    }
    const bool bad = n.live && (pos < 0 || pos >= sh.max_pos);
    if (bad) {
      if (lane == 0) atomicOr(err, kErrIndex);
      pos = 0;
    }
    // out_a = r (x_a pa + other(x_a) qa): the angles times the weights, once for all heads
    float2 pa[VE / 2], qa[VE / 2], pb[VE / 2], qb[VE / 2], wa[VE / 2], wb[VE / 2];
    load_angles<VE, kAdjacent>(cos_sin + pos * sh.rot, pl, sh, n.mine > 0 && !bad, pa, qa, pb, qb);
    R ra = {}, rb = {};
    if (n.mine > 0) {
      const T* w = n.is_q ? wq : wk;
      ra = __ldg(reinterpret_cast<const R*>(w + pl.a));
      rb = __ldg(reinterpret_cast<const R*>(w + pl.b));
    }
    unpack_raw<T, VE>(ra, wa);
    unpack_raw<T, VE>(rb, wb);
#pragma unroll
    for (int e = 0; e < VE / 2; ++e) {
      if constexpr (!kAdjacent) {
        pb[e] = pa[e];
        qb[e] = qa[e];
        qa[e] = neg2(qa[e]);
      }
      pa[e] = __fmul2_rn(pa[e], wa[e]);
      pb[e] = __fmul2_rn(pb[e], wb[e]);
      qa[e] = __fmul2_rn(qa[e], kAdjacent ? swapped(wa[e]) : wb[e]);
      qb[e] = __fmul2_rn(qb[e], kAdjacent ? swapped(wb[e]) : wa[e]);
    }
    T* y = (n.is_q ? q_out : k_out) + (static_cast<int64_t>(n.t) * n.heads + n.h0) * dim;
    if constexpr (kRing) cp_async_wait<1>();
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      if constexpr (kRing) {
        raw[i][0] = raw[i][1] = R{};
        if (i < n.mine) {
          raw[i][0] = reinterpret_cast<const R*>(ring)[slot(stage, i, 0)];
          raw[i][1] = reinterpret_cast<const R*>(ring)[slot(stage, i, 1)];
        }
      }
      float2 a[VE / 2], b[VE / 2], sq = both(0.f);
      unpack_raw<T, VE>(raw[i][0], a);
      unpack_raw<T, VE>(raw[i][1], b);
#pragma unroll
      for (int e = 0; e < VE / 2; ++e) sq = __ffma2_rn(a[e], a[e], __ffma2_rn(b[e], b[e], sq));
      float r = rsqrtf(group_sum(sq.x + sq.y, lanes) / static_cast<float>(dim) + sh.eps);
      if (bad) r = nan_f();
#pragma unroll
      for (int e = 0; e < VE / 2; ++e) {
        float2 ya = __fmul2_rn(a[e], pa[e]), yb = __fmul2_rn(b[e], pb[e]);
        if (pl.turned) {  // not 0 * other: the other may be infinite
          ya = __ffma2_rn(kAdjacent ? swapped(a[e]) : b[e], qa[e], ya);
          yb = __ffma2_rn(kAdjacent ? swapped(b[e]) : a[e], qb[e], yb);
        }
        a[e] = __fmul2_rn(ya, both(r));
        b[e] = __fmul2_rn(yb, both(r));
      }
      if (i < n.mine) {
        store_raw<T, VE>(y + i * dim + pl.a, a);
        store_raw<T, VE>(y + i * dim + pl.b, b);
      }
    }
    stage ^= 1;
    if constexpr (!kRing) break;
  }
  if constexpr (kRing) cp_async_wait<0>();
}

// CTAs [0, q_ctas) go over q's rows, the others over k's; a turn is HPG heads of a token per
// group of lanes. A thread's own vectors come through its own slots of a shared-memory ring
// (cp.async, kBackStages - 1 turns ahead), which takes no registers and no barrier: held in
// registers, loads and sums together left 12 warps an SM. Partial weight gradients to
// partials[cta][dim]: lanes that hold the same elements are added within a warp by halving,
// then the warps in order. Without partials, one CTA to a weight writes its gradient itself.
constexpr int kBackStages = 2;

template <typename T, int VE, int HPG, bool kAdjacent>
__global__ void __launch_bounds__(kVecThreads, 2)
rope_back_vector_pairs(const T* __restrict__ gq, const T* __restrict__ gk,
                       const T* __restrict__ q, const T* __restrict__ k,
                       const T* __restrict__ wq, const T* __restrict__ wk,
                       const float* __restrict__ cos_sin, const int64_t* __restrict__ positions,
                       T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dwq,
                       T* __restrict__ dwk, float* __restrict__ partials, int64_t gq_stride,
                       int64_t gk_stride, int64_t q_stride, int64_t k_stride, int q_ctas,
                       int log_lanes, RopeShape sh, unsigned* err) {
  using R = RawOf<T, VE>;
  // [stage][head][x a, x b, g a, g b][thread]
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float sums[kVecThreads / kWarp][kMaxHeadDim];
  pdl_launch_dependents();
  const int lanes = 1 << log_lanes, lane = threadIdx.x & (lanes - 1);
  const int dim = static_cast<int>(sh.dim);
  const bool is_q = static_cast<int>(blockIdx.x) < q_ctas;
  const int heads = static_cast<int>(is_q ? sh.q_heads : sh.k_heads);
  const uint32_t parts = (heads + HPG - 1) / HPG;
  const int cta = is_q ? blockIdx.x : blockIdx.x - q_ctas;
  const int ctas = is_q ? q_ctas : gridDim.x - q_ctas;
  const T* x0 = is_q ? q : k;
  const T* g0 = is_q ? gq : gk;
  T* dx0 = is_q ? dq : dk;
  const int64_t x_stride = is_q ? q_stride : k_stride, g_stride = is_q ? gq_stride : gk_stride;
  const PairPlace pl = pair_place<VE, kAdjacent>(lane, sh);
  const bool holds = lane * 2 * VE < dim;
  const float inv_d = 1.f / static_cast<float>(dim);

  float2 wa[VE / 2], wb[VE / 2], acc_a[VE / 2] = {}, acc_b[VE / 2] = {};
  R ra = {}, rb = {};
  if (holds) {
    const T* w = is_q ? wq : wk;
    ra = __ldg(reinterpret_cast<const R*>(w + pl.a));
    rb = __ldg(reinterpret_cast<const R*>(w + pl.b));
  }
  unpack_raw<T, VE>(ra, wa);
  unpack_raw<T, VE>(rb, wb);

  // this thread's slot of vector v of head i in a stage
  const auto slot = [&](int stage, int i, int v) {
    return ((stage * HPG + i) * 4 + v) * kVecThreads + static_cast<int>(threadIdx.x);
  };
  const int64_t items = sh.tokens * parts;
  const int64_t step = static_cast<int64_t>(ctas) * (kVecThreads >> log_lanes);
  const int64_t first = static_cast<int64_t>(cta) * (kVecThreads >> log_lanes);
  int64_t ahead = first + (threadIdx.x >> log_lanes);  // the item that is loaded next
  int64_t next_pos = 0;  // its token's position is held until its turn comes
  int64_t held_pos[kBackStages - 1];
  const auto load = [&](int stage) {
    if (ahead < items && holds) {
      const uint32_t t = static_cast<uint32_t>(ahead) / parts;
      const int h0 = static_cast<int>(static_cast<uint32_t>(ahead) - t * parts) * HPG;
      const T* x = x0 + t * x_stride + static_cast<int64_t>(h0) * dim;
      const T* g = g0 + t * g_stride + static_cast<int64_t>(h0) * dim;
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        if (h0 + i >= heads) break;
        const T* src[4] = {x + i * dim + pl.a, x + i * dim + pl.b, g + i * dim + pl.a,
                           g + i * dim + pl.b};
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const uint32_t dst =
              smem_u32(ring) + slot(stage, i, v) * static_cast<uint32_t>(sizeof(R));
          if constexpr (sizeof(R) == 16) cp_async16(dst, src[v], true);
          else cp_async8(dst, src[v], true);
        }
      }
    }
    cp_async_commit();
    next_pos = ahead < items ? positions[static_cast<uint32_t>(ahead) / parts] : 0;
    ahead += step;
  };
#pragma unroll
  for (int i = 0; i < kBackStages - 1; ++i) {
    load(i);
    held_pos[i] = next_pos;
  }

  int stage = 0;
  // every lane of the CTA takes the same number of turns: the shuffles need whole warps
  for (int64_t base = first; base < items; base += step) {
    load(stage == 0 ? kBackStages - 1 : stage - 1);
    const int64_t item = base + (threadIdx.x >> log_lanes);
    const bool live = item < items;
    const uint32_t t = live ? static_cast<uint32_t>(item) / parts : 0;
    const int h0 = live ? static_cast<int>(static_cast<uint32_t>(item) - t * parts) * HPG : 0;
    const int mine = live && holds ? min(HPG, heads - h0) : 0;
    int64_t pos = held_pos[0];
#pragma unroll
    for (int i = 0; i + 1 < kBackStages - 1; ++i) held_pos[i] = held_pos[i + 1];
    held_pos[kBackStages - 2] = next_pos;
    const bool bad = live && (pos < 0 || pos >= sh.max_pos);
    if (bad) {
      if (lane == 0) atomicOr(err, kErrIndex);
      pos = 0;
    }
    float2 ca[VE / 2], sa[VE / 2], cb[VE / 2], sb[VE / 2];
    load_angles<VE, kAdjacent>(cos_sin + pos * sh.rot, pl, sh, mine > 0 && !bad, ca, sa, cb, sb);
    T* dx = dx0 + (static_cast<int64_t>(t) * heads + h0) * dim;
    cp_async_wait<kBackStages - 1>();
    const R* held = reinterpret_cast<const R*>(ring);
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      float2 xa[VE / 2], xb[VE / 2], ya[VE / 2], yb[VE / 2], sq = both(0.f), inner = both(0.f);
      R raw[4] = {};
      if (i < mine) {
#pragma unroll
        for (int v = 0; v < 4; ++v) raw[v] = held[slot(stage, i, v)];
      }
      unpack_raw<T, VE>(raw[0], xa);
      unpack_raw<T, VE>(raw[1], xb);
      unpack_raw<T, VE>(raw[2], ya);
      unpack_raw<T, VE>(raw[3], yb);
#pragma unroll
      for (int e = 0; e < VE / 2; ++e) {
        if (pl.turned) {  // back: the sines change sign
          const float2 ga = ya[e], gb = yb[e];
          if constexpr (!kAdjacent) {
            ya[e] = __ffma2_rn(gb, sa[e], __fmul2_rn(ga, ca[e]));
            yb[e] = __ffma2_rn(neg2(ga), sa[e], __fmul2_rn(gb, ca[e]));
          } else {
            ya[e] = __ffma2_rn(swapped(ga), neg2(sa[e]), __fmul2_rn(ga, ca[e]));
            yb[e] = __ffma2_rn(swapped(gb), neg2(sb[e]), __fmul2_rn(gb, cb[e]));
          }
        }
        sq = __ffma2_rn(xa[e], xa[e], __ffma2_rn(xb[e], xb[e], sq));
        inner = __ffma2_rn(__fmul2_rn(ya[e], wa[e]), xa[e],
                           __ffma2_rn(__fmul2_rn(yb[e], wb[e]), xb[e], inner));
      }
      const float2 sums2 = group_sum2(make_float2(sq.x + sq.y, inner.x + inner.y), lanes);
      float r = rsqrtf(sums2.x * inv_d + sh.eps);
      if (bad) r = nan_f();
      // dx = r dy w - x r^2 mean(dn x r) with mean(dn x r) = r mean(dn x)
      const float m = sums2.y * inv_d * r;
      const float2 r2 = both(r), mr = both(-m * r);
#pragma unroll
      for (int e = 0; e < VE / 2; ++e) {
        xa[e] = __fmul2_rn(xa[e], r2);
        xb[e] = __fmul2_rn(xb[e], r2);
        if (i < mine) {
          acc_a[e] = __ffma2_rn(ya[e], xa[e], acc_a[e]);
          acc_b[e] = __ffma2_rn(yb[e], xb[e], acc_b[e]);
        }
        xa[e] = __ffma2_rn(xa[e], mr, __fmul2_rn(__fmul2_rn(ya[e], wa[e]), r2));
        xb[e] = __ffma2_rn(xb[e], mr, __fmul2_rn(__fmul2_rn(yb[e], wb[e]), r2));
      }
      if (i < mine) {
        store_raw<T, VE>(dx + i * dim + pl.a, xa);
        store_raw<T, VE>(dx + i * dim + pl.b, xb);
      }
    }
    stage = stage + 1 == kBackStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  const int warp = threadIdx.x / kWarp;
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    float va = e % 2 ? acc_a[e / 2].y : acc_a[e / 2].x;
    float vb = e % 2 ? acc_b[e / 2].y : acc_b[e / 2].x;
    for (int o = lanes; o < kWarp; o <<= 1) {
      va += __shfl_xor_sync(kFull, va, o);
      vb += __shfl_xor_sync(kFull, vb, o);
    }
    if ((threadIdx.x & (kWarp - 1)) < lanes && holds) {
      sums[warp][pl.a + e] = va;
      sums[warp][pl.b + e] = vb;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < dim; i += kVecThreads) {
    float total = 0.f;
#pragma unroll
    for (int j = 0; j < kVecThreads / kWarp; ++j) total += sums[j][i];
    if (partials != nullptr) {
      partials[static_cast<int64_t>(blockIdx.x) * dim + i] = total;
    } else {  // the only CTA of its weight; alone, the other has no rows
      (is_q ? dwq : dwk)[i] = from_f<T>(total);
      if (gridDim.x == 1) (is_q ? dwk : dwq)[i] = from_f<T>(0.f);
    }
  }
}

// ------------------------------------------------------------------ weight gradients

// Partials of one weight: `count` rows of dim floats, `stride` apart.
struct Partials {
  const float* at;
  int64_t count, stride;
};

// dw[i] = sum of the partials: every 32nd one by one row of threads, then the 32 rows in
// order, so the same bits every time.
constexpr int kFinishRows = 32;

template <typename T>
__global__ void __launch_bounds__(kWarp * kFinishRows)
rope_weight_finish(Partials pq, Partials pk, int dim, T* dwq, T* dwk) {
  __shared__ float part[kFinishRows][kWarp + 1];
  const Partials p = blockIdx.y == 0 ? pq : pk;
  const int lane = threadIdx.x & (kWarp - 1), slice = threadIdx.x / kWarp;
  const int i = blockIdx.x * kWarp + lane;
  pdl_wait_primary();
  float s = 0.f;
  if (i < dim) {
#pragma unroll 4
    for (int64_t c = slice; c < p.count; c += kFinishRows) s += p.at[c * p.stride + i];
  }
  part[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && i < dim) {
    s = 0.f;
    for (int j = 0; j < kFinishRows; ++j) s += part[j][lane];
    (blockIdx.y == 0 ? dwq : dwk)[i] = from_f<T>(s);
  }
}

// ------------------------------------------------------------------ launch

// CTAs of the backward's first kernel per weight (each writes one partial).
int64_t back_ctas(const RopeShape& sh, int sms) {
  const int64_t rows = sh.tokens * std::max(sh.q_heads, sh.k_heads);
  return std::max<int64_t>(1, std::min<int64_t>(cdiv(rows, kWarpsPerCta), int64_t{4} * sms));
}

uintptr_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Elements of the vectors that variant 1 takes this call in, 0 where it does not: 16 bytes,
// or 8 for 16-bit types (a rotated part of 40 elements, say, is no whole number of pairs of
// 16-byte vectors). `all` holds the or of all addresses, `strides` of all token strides.
template <typename T>
int vector_elements(const RopeShape& sh, uintptr_t all, int64_t strides, const float* cos_sin) {
  if (addr(cos_sin) % 16 != 0) return 0;
  for (int ve = Vec<T>::kN; ve >= 4; ve /= 2) {
    if (sh.rot % (2 * ve) == 0 && (sh.dim - sh.rot) % (2 * ve) == 0 &&
        all % (ve * sizeof(T)) == 0 && (sh.tokens < 2 || strides % ve == 0))
      return ve;
  }
  return 0;
}

int lanes_log2(int64_t pairs) {
  int log = 0;
  while ((int64_t{1} << log) < pairs) ++log;
  return log;
}

template <typename T, int VE, int HPG, bool kRing>
int launch_pairs(const T* q, const T* k, const T* wq, const T* wk, const float* cos_sin,
                 const int64_t* positions, T* q_out, T* k_out, int64_t q_stride,
                 int64_t k_stride, const RopeShape& sh, unsigned* err, cudaStream_t s) {
  const int log = lanes_log2(sh.dim / (2 * VE));
  const int64_t items = sh.tokens * (cdiv(sh.q_heads, HPG) + cdiv(sh.k_heads, HPG));
  int64_t ctas = cdiv(items << log, kRopeThreads);
  auto* kernel = sh.interleaved ? rope_vector_pairs<T, VE, HPG, true, kRing>
                                : rope_vector_pairs<T, VE, HPG, false, kRing>;
  int smem = 0;
  if constexpr (kRing) {
    const void* fn = reinterpret_cast<const void*>(kernel);
    smem = kForwardStages * HPG * 2 * kRopeThreads * VE * static_cast<int>(sizeof(T));
    int occ = 0;
    if (int rc = ensure_dyn_smem(fn, smem)) return rc;
    if (int rc = occupancy_blocks(fn, kRopeThreads, smem, &occ)) return rc;
    ctas = std::min(ctas, int64_t{occ} * sm_count());
  }
  kernel<<<static_cast<unsigned>(ctas), kRopeThreads, smem, s>>>(
      q, k, wq, wk, cos_sin, positions, q_out, k_out, q_stride, k_stride, log, sh, err);
  KPB_LAUNCHED("qk_norm_rope vector pairs");
  return KPB_OK;
}

// Four heads to a turn once that still gives every SM 1024 threads; one where rows are few.
// Many rows of 16-bit values go through the ring (16384 tokens x 40 heads x 128: 59 us, 68
// read into registers); fp32 vectors hold half the values, leave more threads room and do
// better without it (4000 tokens: 28 us against 30).
template <typename T, int VE>
int dispatch_pairs(const T* q, const T* k, const T* wq, const T* wk, const float* cos_sin,
                   const int64_t* positions, T* q_out, T* k_out, int64_t q_stride,
                   int64_t k_stride, const RopeShape& sh, unsigned* err, cudaStream_t s) {
  const int64_t threads = sh.tokens * (sh.q_heads + sh.k_heads) << lanes_log2(sh.dim / (2 * VE));
  if (threads >= int64_t{4} * 1024 * sm_count())
    return launch_pairs<T, VE, 4, sizeof(T) == 2>(q, k, wq, wk, cos_sin, positions, q_out, k_out,
                                                  q_stride, k_stride, sh, err, s);
  return launch_pairs<T, VE, 1, false>(q, k, wq, wk, cos_sin, positions, q_out, k_out, q_stride,
                                       k_stride, sh, err, s);
}

template <typename T>
int launch(int variant, const T* q, const T* k, const T* wq, const T* wk, const float* cos_sin,
           const int64_t* positions, T* q_out, T* k_out, int64_t q_stride, int64_t k_stride,
           const RopeShape& sh, unsigned* err, cudaStream_t s) {
  if (variant == 1) {
    const int ve = vector_elements<T>(
        sh, addr(q) | addr(k) | addr(wq) | addr(wk) | addr(q_out) | addr(k_out),
        q_stride | k_stride, cos_sin);
    if (ve == Vec<T>::kN)
      return dispatch_pairs<T, Vec<T>::kN>(q, k, wq, wk, cos_sin, positions, q_out, k_out,
                                           q_stride, k_stride, sh, err, s);
    if (ve == 4)
      return dispatch_pairs<T, 4>(q, k, wq, wk, cos_sin, positions, q_out, k_out, q_stride,
                                  k_stride, sh, err, s);
  }
  const int64_t rows = sh.tokens * (sh.q_heads + sh.k_heads);
  rope_warp_row<T><<<static_cast<unsigned>(cdiv(rows, kWarpsPerCta)), kWarpsPerCta * kWarp, 0, s>>>(
      q, k, wq, wk, cos_sin, positions, q_out, k_out, q_stride, k_stride, sh, err);
  KPB_LAUNCHED("qk_norm_rope");
  return KPB_OK;
}

template <typename T>
int finish_weights(const Partials& pq, const Partials& pk, int dim, T* dwq, T* dwk, bool dependent,
                   cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(cdiv(dim, kWarp)), 2);
  cfg.blockDim = dim3(kWarp * kFinishRows);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  KPB_CUDA(cudaLaunchKernelEx(&cfg, rope_weight_finish<T>, pq, pk, dim, dwq, dwk));
  return KPB_OK;
}

template <typename T, int VE>
int launch_back_pairs(const T* gq, const T* gk, const T* q, const T* k, const T* wq, const T* wk,
                      const float* cos_sin, const int64_t* positions, T* dq, T* dk, T* dwq,
                      T* dwk, int64_t gq_stride, int64_t gk_stride, int64_t q_stride,
                      int64_t k_stride, const RopeShape& sh, float* partials, unsigned* err,
                      cudaStream_t s) {
  constexpr int HPG = 2;
  const int dim = static_cast<int>(sh.dim), log = lanes_log2(dim / (2 * VE));
  auto* kernel = sh.interleaved ? rope_back_vector_pairs<T, VE, HPG, true>
                                : rope_back_vector_pairs<T, VE, HPG, false>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  constexpr int kSmem = kBackStages * HPG * 4 * kVecThreads * VE * static_cast<int>(sizeof(T));
  int occ = 0;
  if (int rc = ensure_dyn_smem(fn, kSmem)) return rc;
  if (int rc = occupancy_blocks(fn, kVecThreads, kSmem, &occ)) return rc;
  // one wave, shared out by the heads; no more CTAs than there is work for, nor than partials
  const int64_t wave = int64_t{occ} * sm_count(), most = back_ctas(sh, sm_count());
  const int64_t heads = sh.q_heads + sh.k_heads;
  // two turns of one CTA take less time than a second kernel
  const auto threads_of = [&](int64_t h) { return sh.tokens * cdiv(h, HPG) << log; };
  const bool alone = std::max(threads_of(sh.q_heads), threads_of(sh.k_heads)) <= 2 * kVecThreads;
  const auto ctas_of = [&](int64_t h) {
    if (h == 0 || sh.tokens == 0) return int64_t{0};
    if (alone) return int64_t{1};
    return std::max<int64_t>(
        1, std::min({cdiv(threads_of(h), kVecThreads), wave * h / heads, most}));
  };
  const int64_t nq = ctas_of(sh.q_heads), nk = ctas_of(sh.k_heads);
  if (nq + nk > 0) {
    kernel<<<static_cast<unsigned>(nq + nk), kVecThreads, kSmem, s>>>(
        gq, gk, q, k, wq, wk, cos_sin, positions, dq, dk, dwq, dwk, alone ? nullptr : partials,
        gq_stride, gk_stride, q_stride, k_stride, static_cast<int>(nq), log, sh, err);
    KPB_LAUNCHED("qk_norm_rope_backward vector pairs");
    if (alone) return KPB_OK;
  }
  return finish_weights<T>({partials, nq, dim}, {partials + nq * dim, nk, dim}, dim, dwq, dwk,
                           nq + nk > 0, s);
}

template <typename T>
int launch_back(int variant, const T* gq, const T* gk, const T* q, const T* k, const T* wq,
                const T* wk, const float* cos_sin, const int64_t* positions, T* dq, T* dk, T* dwq,
                T* dwk, int64_t gq_stride, int64_t gk_stride, int64_t q_stride, int64_t k_stride,
                const RopeShape& sh, float* partials, unsigned* err, cudaStream_t s) {
  if (variant == 1) {
    const int ve = vector_elements<T>(
        sh, addr(gq) | addr(gk) | addr(q) | addr(k) | addr(wq) | addr(wk) | addr(dq) | addr(dk),
        gq_stride | gk_stride | q_stride | k_stride, cos_sin);
    if (ve == Vec<T>::kN)
      return launch_back_pairs<T, Vec<T>::kN>(gq, gk, q, k, wq, wk, cos_sin, positions, dq, dk,
                                              dwq, dwk, gq_stride, gk_stride, q_stride, k_stride,
                                              sh, partials, err, s);
    if (ve == 4)
      return launch_back_pairs<T, 4>(gq, gk, q, k, wq, wk, cos_sin, positions, dq, dk, dwq, dwk,
                                     gq_stride, gk_stride, q_stride, k_stride, sh, partials, err,
                                     s);
  }
  const int64_t ctas = back_ctas(sh, sm_count());
  rope_back_warp_row<T><<<static_cast<unsigned>(ctas), kWarpsPerCta * kWarp, 0, s>>>(
      gq, gk, q, k, wq, wk, cos_sin, positions, dq, dk, partials, gq_stride, gk_stride, q_stride,
      k_stride, sh, err);
  KPB_LAUNCHED("qk_norm_rope_backward");
  return finish_weights<T>({partials, ctas, 2 * sh.dim}, {partials + sh.dim, ctas, 2 * sh.dim},
                           static_cast<int>(sh.dim), dwq, dwk, false, s);
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
#define KPB_ROPE(T)                                                                \
  launch<T>(variant, static_cast<const T*>(q), static_cast<const T*>(k),          \
            static_cast<const T*>(wq), static_cast<const T*>(wk), cos_sin,        \
            positions, static_cast<T*>(q_out), static_cast<T*>(k_out), q_stride,  \
            k_stride, sh, err, s)
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
  launch_back<T>(variant, static_cast<const T*>(gq), static_cast<const T*>(gk),                \
                 static_cast<const T*>(q),                                                     \
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
