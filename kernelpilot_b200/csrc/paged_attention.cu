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
//   variant 1  the keys of all sequences split evenly over one wave of CTAs, whatever the
//              lengths are. A unit of work is 64 keys of one row, a row being a (sequence,
//              key head, tile of its query heads); CTA c of W takes units c * total / W to
//              (c + 1) * total / W, found from the lengths on the device, so one captured
//              call serves any lengths. A row that lies in one CTA is finished there; one
//              that several CTAs share leaves a partial (maximum, sum, weighted values) per
//              CTA, joined in CTA order by a second kernel (a programmatic dependent).
//              Each of a CTA's four warps takes 16 of a unit's keys and streams its own
//              keys and values, so no barrier stands between a load and its use; the warps
//              meet once per row. Two ways to the products:
//                split_mma   fp16 / bf16 q, rows a multiple of 16 bytes on 16-byte
//                            boundaries: cp.async into a swizzled ring per warp, mma.sync
//                split_simt  everything else (fp32, odd head dims, odd bases)
#include <algorithm>

#include "kp_kv_cache.cuh"
#include "kp_sm100.cuh"

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

// ------------------------------------------------------------------ variant 1: the split

constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = kSplitWarps * kWarp;

// How rows and units are laid out: a unit is `unit` keys of a row; rows of a sequence are (key head, tile of `tile_heads`
// query heads), tiles innermost; a partial has tile_heads x (pitch) floats: pitch - 4
// weighted values, then maximum and sum.
struct SplitShape {
  int64_t rows;      // rows per sequence
  int tiles;         // tiles of query heads per key head
  int group;         // query heads per key head
  int tile_heads;
  int pitch;
  int unit_log;      // log2 of the keys per unit
  int64_t* bases;    // workspace: units before each sequence (batch), then their total
  float* partials;   // workspace: [cta][2][tile_heads][pitch]
};

// Units of a row of n keys.
__device__ __forceinline__ int units_of(int64_t n, const SplitShape& sp) {
  return static_cast<int>((n + (1 << sp.unit_log) - 1) >> sp.unit_log);
}

__device__ __forceinline__ int64_t first_unit(int64_t cta, int64_t ctas, int64_t total) {
  return cta * total / ctas;
}

// The CTA that unit u falls to (the inverse of first_unit).
__device__ __forceinline__ int64_t cta_of_unit(int64_t u, int64_t ctas, int64_t total) {
  return ((u + 1) * ctas - 1) / total;
}

// A place in the list of units: sequence, row, block of keys.
struct UnitPlace {
  int64_t b, row;
  int blk, blocks;  // block within the row, blocks of the row
  int n;            // keys of the sequence

  __device__ __forceinline__ void next(const int* __restrict__ seq_lens, const PagedShape& sh,
                                       const SplitShape& sp, unsigned* err) {
    if (++blk < blocks) return;
    blk = 0;
    if (++row < sp.rows) return;
    row = 0;
    do {
      ++b;
      n = b < sh.batch ? static_cast<int>(keys_of(seq_lens, b, sh, err)) : 1;
      blocks = units_of(n, sp);
    } while (blocks == 0);
  }
};

// This CTA's units [*begin, *end) and the place of the first. Every thread calls it;
// `scratch` holds kSplitWarps + 3 int64. CTA 0 leaves bases and total in the workspace.
__device__ __forceinline__ UnitPlace find_units(const int* __restrict__ seq_lens,
                                                const PagedShape& sh, const SplitShape& sp,
                                                int64_t* scratch, int64_t* begin, int64_t* end,
                                                unsigned* err) {
  const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
  const int64_t per = (sh.batch + kSplitThreads - 1) / kSplitThreads;
  const int64_t b0 = min(sh.batch, threadIdx.x * per), b1 = min(sh.batch, b0 + per);
  int64_t mine = 0;
  for (int64_t b = b0; b < b1; ++b)
    mine += units_of(keys_of(seq_lens, b, sh, err), sp) * sp.rows;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < kWarp; o <<= 1) {
    const int64_t v = __shfl_up_sync(kFull, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == kWarp - 1) scratch[warp] = upto;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kSplitWarps; ++w) {
    if (w < warp) upto += scratch[w];
    total += scratch[w];
  }
  int64_t base = upto - mine;
  // no more CTAs than units: every CTA of a shared row then has a part of it
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total), cta = blockIdx.x;
  *begin = cta < ctas ? first_unit(cta, ctas, total) : 0;
  *end = cta < ctas ? first_unit(cta + 1, ctas, total) : 0;
  const bool here = *begin < *end && *begin >= base && *begin < upto;
  if (blockIdx.x == 0 || here) {
    for (int64_t b = b0; b < b1; ++b) {
      const int64_t units = units_of(keys_of(seq_lens, b, sh, err), sp) * sp.rows;
      if (blockIdx.x == 0) sp.bases[b] = base;
      if (here && *begin >= base && *begin < base + units) {
        scratch[kSplitWarps] = b;
        scratch[kSplitWarps + 1] = base;
      }
      base += units;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) sp.bases[sh.batch] = total;
  }
  __syncthreads();
  UnitPlace p = {};
  if (*begin < *end) {
    p.b = scratch[kSplitWarps];
    const int64_t in = *begin - scratch[kSplitWarps + 1];
    p.n = static_cast<int>(keys_of(seq_lens, p.b, sh, err));
    p.blocks = units_of(p.n, sp);
    p.row = in / p.blocks;
    p.blk = static_cast<int>(in - p.row * p.blocks);
  }
  __syncthreads();
  return p;
}

// Zeros for the sequences without keys, strided over the CTAs.
template <typename T>
__device__ __forceinline__ void zero_empty(T* __restrict__ o, const int* __restrict__ seq_lens,
                                           const PagedShape& sh, unsigned* err) {
  const int64_t row = sh.q_heads * sh.lay.dim;
  for (int64_t b = blockIdx.x; b < sh.batch; b += gridDim.x) {
    if (keys_of(seq_lens, b, sh, err) != 0) continue;
    for (int64_t i = threadIdx.x; i < row; i += kSplitThreads) o[b * row + i] = from_f<T>(0.f);
  }
}

// Joins the warps' parts of the segment that ends here (maximum s_m and sum s_l,
// [warp][head]; weighted values s_o, [warp][head - h0][pitch], of heads h0 to h0 + held of
// the tile) and writes it: the output where the segment is a whole row, else partial `slot`
// of this CTA.
template <typename T>
__device__ __forceinline__ void write_segment(const float* s_m, const float* s_l,
                                              const float* s_o, int h0, int held,
                                              const UnitPlace& p, bool whole, int slot,
                                              T* __restrict__ o, const PagedShape& sh,
                                              const SplitShape& sp) {
  const int64_t hk = p.row / sp.tiles;
  const int first = static_cast<int>(p.row - hk * sp.tiles) * sp.tile_heads;
  const int h1 = min(h0 + held, sp.group - first);
  const int dim = static_cast<int>(sh.lay.dim);
  for (int h = h0; h < h1; ++h) {
    float f[kSplitWarps], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) top = fmaxf(top, s_m[w * sp.tile_heads + h]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      f[w] = ex2f(s_m[w * sp.tile_heads + h] - base);
      sum = fmaf(f[w], s_l[w * sp.tile_heads + h], sum);
    }
    float* part = sp.partials +
                  ((static_cast<int64_t>(blockIdx.x) * 2 + slot) * sp.tile_heads + h) * sp.pitch;
    for (int i = threadIdx.x; i < dim; i += kSplitThreads) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kSplitWarps; ++w)
        v = fmaf(f[w], s_o[(w * held + h - h0) * sp.pitch + i], v);
      if (whole) {
        o[(p.b * sh.q_heads + hk * sp.group + first + h) * dim + i] = from_f<T>(v / sum);
      } else {
        part[i] = v;
      }
    }
    if (!whole && threadIdx.x == 0) {
      part[sp.pitch - 4] = top;
      part[sp.pitch - 3] = sum;
    }
  }
}

// One CTA per row that several CTAs share, one warp per query head at a time, lanes
// strided over the values: out = sum_c f_c O_c / sum_c f_c l_c over the row's partials in
// CTA order, f_c = 2^(m_c - max m). `ctas` is the first kernel's grid.
constexpr int kJoinWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * kWarp)
join_rows(const int* __restrict__ seq_lens, T* __restrict__ o, PagedShape sh, SplitShape sp,
          int64_t ctas, unsigned* err) {
  const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
  const int64_t b = blockIdx.x / sp.rows, row = blockIdx.x - b * sp.rows;
  const int64_t blocks = units_of(keys_of(seq_lens, b, sh, err), sp);
  pdl_wait_primary();
  const int64_t total = sp.bases[sh.batch], base = sp.bases[b];
  if (blocks < 2) return;
  ctas = min(ctas, total);
  const int64_t u0 = base + row * blocks;
  const int64_t c0 = cta_of_unit(u0, ctas, total), c1 = cta_of_unit(u0 + blocks - 1, ctas, total);
  if (c0 == c1) return;
  const int64_t hk = row / sp.tiles;
  const int first = static_cast<int>(row - hk * sp.tiles) * sp.tile_heads;
  const int heads = min(sp.tile_heads, sp.group - first);
  const int dim = static_cast<int>(sh.lay.dim);
  const int count = static_cast<int>(c1 - c0) + 1;
  // only the first CTA's segment may start inside its range (slot 1)
  const int slot0 = u0 > first_unit(c0, ctas, total) ? 1 : 0;
  const int64_t step = static_cast<int64_t>(2) * sp.tile_heads * sp.pitch;
  for (int h = warp; h < heads; h += kJoinWarps) {
    const float* p0 = sp.partials + ((c0 * 2 + slot0) * sp.tile_heads + h) * sp.pitch;
    const float* rest = sp.partials + (c0 * 2 * sp.tile_heads + h) * sp.pitch;
    float top = -INFINITY;
    for (int c = lane; c < count; c += kWarp)
      top = fmaxf(top, (c == 0 ? p0 : rest + c * step)[sp.pitch - 4]);
    top = warp_max(top);
    if (top == -INFINITY) top = 0.f;
    float sum = 0.f, acc[kPerLane] = {};
#pragma unroll 4
    for (int c = 0; c < count; ++c) {
      const float* p = c == 0 ? p0 : rest + c * step;
      const float f = ex2f(p[sp.pitch - 4] - top);
      sum = fmaf(f, p[sp.pitch - 3], sum);
#pragma unroll
      for (int e = 0; e < kPerLane; ++e) {
        const int i = lane + e * kWarp;
        if (i < dim) acc[e] = fmaf(f, p[i], acc[e]);
      }
    }
    T* out = o + (b * sh.q_heads + hk * sp.group + first + h) * dim;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) {
      const int i = lane + e * kWarp;
      if (i < dim) out[i] = from_f<T>(acc[e] / sum);
    }
  }
}

// The cache row of key `pos` of sequence b under key head hk, in elements; -1 past the
// last key, -2 (and kErrIndex) for a page outside the cache.
__device__ __forceinline__ int64_t key_row(const int* __restrict__ table, int64_t b, int pos,
                                           int n, int64_t hk, const PagedShape& sh,
                                           int64_t* scale_at, unsigned* err) {
  if (pos >= n) return -1;
  const int size = static_cast<int>(sh.lay.page_size);
  const int at = pos / size;
  const int64_t page = table[b * sh.table_stride + at];
  if (page < 0 || page >= sh.lay.num_pages) {
    atomicOr(err, kErrIndex);
    return -2;
  }
  *scale_at = sh.lay.scale(page, hk, pos - at * size);
  return sh.lay.row(page, hk, pos - at * size);
}

// ------------------------------------------------------------------ variant 1: split_simt

constexpr int kSimtUnit = 64;

// Lanes are strided over a row's elements (E each); a warp takes 4 keys at a time and HG
// query heads: 4 * HG products, summed over the lanes by halving, so that each lane ends
// with the score of one (key, head).
template <typename T, typename C, int E, int HG>
__global__ void __launch_bounds__(kSplitThreads)
split_simt(const T* __restrict__ q, const C* __restrict__ k_cache, const C* __restrict__ v_cache,
           const int* __restrict__ table, const int* __restrict__ seq_lens,
           const float* __restrict__ k_scale, const float* __restrict__ v_scale,
           T* __restrict__ o, PagedShape sh, SplitShape sp, unsigned* err) {
  constexpr int kKeys = 4, kWarpKeys = kSimtUnit / kSplitWarps;
  constexpr int kSums = kKeys * HG;
  constexpr int kLog = kSums == 32 ? 5 : kSums == 16 ? 4 : kSums == 8 ? 3 : 2;
  constexpr int kSpread = 5 - kLog;  // 2^kSpread neighbouring lanes hold the same sum
  constexpr bool kQuant = std::is_same_v<C, uint8_t>;
  constexpr int kPitch = E * kWarp + 4;
  __shared__ float s_m[kSplitWarps * HG], s_l[kSplitWarps * HG];
  __shared__ float s_o[kSplitWarps * HG * kPitch];
  __shared__ int64_t scratch[kSplitWarps + 2];
  const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
  const int dim = static_cast<int>(sh.lay.dim);
  pdl_launch_dependents();
  zero_empty(o, seq_lens, sh, err);
  int64_t u, end;
  UnitPlace p = find_units(seq_lens, sh, sp, scratch, &u, &end, err);
  const int my_key = (lane >> kSpread) / HG;

  float qr[HG][E], acc[HG][E], m = -INFINITY, l = 0.f;
  bool fresh = true, whole_start = p.blk == 0;
  int slot = 0;
  for (; u < end; ++u) {
    const int64_t hk = p.row / sp.tiles;
    const int first = static_cast<int>(p.row - hk * sp.tiles) * HG;
    if (fresh) {
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const T* qh = q + p.b * sh.q_stride + (hk * sp.group + first + h) * dim;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = lane + e * kWarp;
          qr[h][e] = i < dim && first + h < sp.group ? to_f(qh[i]) * (sh.scale * kLog2e) : 0.f;
          acc[h][e] = 0.f;
        }
      }
      m = -INFINITY;
      l = 0.f;
      fresh = false;
    }
    const int key0 = p.blk * kSimtUnit + warp * kWarpKeys;
    int64_t my_scale = 0;
    const int64_t my_row = lane < kWarpKeys
                               ? key_row(table, p.b, key0 + lane, p.n, hk, sh, &my_scale, err)
                               : -1;
    if (__any_sync(kFull, my_row == -2)) l = nan_f();
    float ks = 1.f, vs = 1.f;
    if constexpr (kQuant) {
      if (my_row >= 0) {
        ks = k_scale[my_scale];
        vs = v_scale[my_scale];
      }
    }
#pragma unroll 1
    for (int j = 0; j < kWarpKeys && key0 + j < p.n; j += kKeys) {
      float kv[kKeys][E], vv[kKeys][E];
      int64_t row[kKeys];
#pragma unroll
      for (int k = 0; k < kKeys; ++k) row[k] = __shfl_sync(kFull, my_row, j + k);
#pragma unroll
      for (int k = 0; k < kKeys; ++k) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = lane + e * kWarp;
          const bool in = i < dim && row[k] >= 0;
          kv[k][e] = in ? cache_value(k_cache + row[k], i, 1.f) : 0.f;
          vv[k][e] = in ? cache_value(v_cache + row[k], i, 1.f) : 0.f;
        }
      }
      float s[kSums];
#pragma unroll
      for (int k = 0; k < kKeys; ++k) {
#pragma unroll
        for (int h = 0; h < HG; ++h) {
          float d = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) d = fmaf(qr[h][e], kv[k][e], d);
          s[k * HG + h] = d;
        }
      }
#pragma unroll
      for (int step = 0; step < kLog; ++step) {
        const int off = 16 >> step, half = kSums >> (step + 1);
        const bool upper = lane & off;
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const float keep = upper ? s[i + half] : s[i];
          const float send = upper ? s[i] : s[i + half];
          s[i] = keep + __shfl_xor_sync(kFull, send, off);
        }
      }
      float score = s[0];
#pragma unroll
      for (int off = (1 << kSpread) >> 1; off > 0; off >>= 1)
        score += __shfl_xor_sync(kFull, score, off);
      if constexpr (kQuant) score *= __shfl_sync(kFull, ks, j + my_key);
      const int64_t key_at = __shfl_sync(kFull, my_row, j + my_key);  // below 0 past the end
      if (key_at < 0) score = -INFINITY;
      float top = score;
#pragma unroll
      for (int off = HG << kSpread; off < kWarp; off <<= 1)
        top = fmaxf(top, __shfl_xor_sync(kFull, top, off));
      const float m_new = fmaxf(m, top);
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m - base);
      float w = exp2f(score - base);
      l = fmaf(l, alpha, w);
      m = m_new;
      if (__any_sync(kFull, alpha != 1.f)) {
#pragma unroll
        for (int h = 0; h < HG; ++h) {
          const float a = __shfl_sync(kFull, alpha, h << kSpread);
#pragma unroll
          for (int e = 0; e < E; ++e) acc[h][e] *= a;
        }
      }
      if constexpr (kQuant) w *= __shfl_sync(kFull, vs, j + my_key);
#pragma unroll
      for (int k = 0; k < kKeys; ++k) {
#pragma unroll
        for (int h = 0; h < HG; ++h) {
          const float pk = __shfl_sync(kFull, w, (k * HG + h) << kSpread);
#pragma unroll
          for (int e = 0; e < E; ++e) acc[h][e] = fmaf(pk, vv[k][e], acc[h][e]);
        }
      }
    }
    const bool row_ends = p.blk + 1 == p.blocks;
    if (row_ends || u + 1 == end) {
      float sum = l;
#pragma unroll
      for (int off = HG << kSpread; off < kWarp; off <<= 1)
        sum += __shfl_xor_sync(kFull, sum, off);
      const int h = (lane >> kSpread) % HG;
      if (lane == h << kSpread) {
        s_m[warp * HG + h] = m;
        s_l[warp * HG + h] = sum;
      }
#pragma unroll
      for (int hh = 0; hh < HG; ++hh) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          s_o[(warp * HG + hh) * kPitch + lane + e * kWarp] = acc[hh][e];
      }
      __syncthreads();
      write_segment(s_m, s_l, s_o, 0, HG, p, whole_start && row_ends, slot, o, sh, sp);
      __syncthreads();
      fresh = true;
      whole_start = true;
      slot = 1;
    }
    p.next(seq_lens, sh, sp, err);
  }
}

// ------------------------------------------------------------------ variant 1: split_mma

// Four 8 x 8 blocks of 16-bit units; lane l gives the address of row l % 8 of block l / 8.
template <bool kTrans>
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (kTrans) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  } else {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  }
}

// The 8 x 8 block of 16-bit values held as a fragment, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// d (16 x 8 fp32) += a (16 x 16) b (16 x 8).
template <typename M>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<M, __half>) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
                 "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
                 "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// Weights w >= 0 as a pair of M (x in the low half) cut towards zero, and as *rest what that
// leaves. The rest is never 0 beside a weight that is not: an infinite value times the pair
// is then an infinity, not infinity * 0.
template <typename M>
__device__ __forceinline__ uint32_t split_weights(float x, float y, uint32_t* rest) {
  constexpr float kTiny = 1.f / (1 << 24);
  uint32_t hi;
  float2 f;
  if constexpr (std::is_same_v<M, __half>) {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
    f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  } else {
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
    f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&hi));
  }
  const float rx = fmaxf(x - f.x, fminf(x, kTiny)), ry = fmaxf(y - f.y, fminf(y, kTiny));
  if constexpr (std::is_same_v<M, __half>) {
    const __half2 v = __floats2half2_rn(rx, ry);
    *rest = *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(rx, ry);
    *rest = *reinterpret_cast<const uint32_t*>(&v);
  }
  return hi;
}

// Weights are held times 2^14 (the maximum's weight is 16384): fp16 then keeps its full
// fraction down to 2^-28 of the largest weight and something down to 2^-38.
constexpr float kWeightBits = 14.f;

// Two e4m3 codes (the low 16 bits) as a pair of fp16, exactly.
__device__ __forceinline__ uint32_t codes_to_half(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | static_cast<uint32_t>(h.y) << 16;
}

// Byte offset of 16-byte chunk `ch` of row `row` in a tile of rows of kRow bytes, chunks
// exchanged so that eight rows' equal chunks lie in different banks.
template <int kRow>
__device__ __forceinline__ uint32_t tile_at(int row, int ch) {
  if constexpr (kRow >= 128) {
    return static_cast<uint32_t>(row * kRow + ((ch ^ (row & 7)) << 4));
  } else {  // two rows to a 128-byte line
    return static_cast<uint32_t>(row * kRow + ((ch ^ ((row >> 1) & 3)) << 4));
  }
}

// Shared memory of one CTA: kStages x (keys, values, scales) per warp, then the warps'
// meeting place, kMeetHeads heads at a time. A warp takes 32 keys at a time where a row is
// 128 bytes at most, else 16. As many stages as let three CTAs share an SM, two at least
// and four at most; with two that do not fit, two CTAs or one.
constexpr int kMeetHeads = 4;

template <typename C, int DP, int NT>
struct MmaPlan {
  static constexpr bool kQuant = std::is_same_v<C, uint8_t>;
  static constexpr int kRow = DP * static_cast<int>(sizeof(C));
  static constexpr int kKeys = kRow <= 128 && DP * NT <= 128 ? 32 : 16;
  static constexpr int kUnit = kSplitWarps * kKeys;
  static constexpr int kTile = kKeys * kRow;
  static constexpr int kStage = 2 * kTile + (kQuant ? 2 * kKeys * 4 : 0);
  static constexpr int kHeads = 8 * NT;
  static constexpr int kPitch = DP + 4;
  static constexpr int kMeet = kSplitWarps * (2 * kHeads + kMeetHeads * kPitch) * 4 + 64;
  static constexpr int kThirdSm = 228 * 1024 / 3 - 1024;
  static constexpr int kFit = (kThirdSm - kMeet) / (kSplitWarps * kStage);
  static constexpr int kStages = kFit < 2 ? 2 : kFit > 4 ? 4 : kFit;
  static constexpr int kSmem = kSplitWarps * kStages * kStage + kMeet;
};

// Rows of the cache as the loader holds them: 16-byte units from the cache's start, in 32
// bits (mma_takes bounds the cache), or one of two marks.
constexpr uint32_t kNoRow = 0xffffffffu;   // past the last key
constexpr uint32_t kBadRow = 0xfffffffeu;  // in a page outside the cache

// T: q and o. C: the cache (T, or e4m3 codes). DP: head dim, padded with zeros. NT: tiles
// of 8 query heads.
// Per 16 keys a warp computes S^T = K Q^T (keys x heads) with K from shared memory as the
// first operand, so that a group of 8 heads fills a product and none is padded, turns the
// weights' fragments over (movmatrix) and adds O^T += V^T P^T (elements x heads). The
// weights enter as two 16-bit parts (split_weights), so that they carry 2^-15 of themselves
// (bf16) or 2^-21 (fp16); the second product is a small part of the time that loading takes.
// e4m3: codes become fp16 in registers, q is scaled by a power of two to [1, 2) (exact) and
// the key's scale multiplies its score. The value's scale goes into the weight in log2
// before the exponential, with a maximum of its own, so that a weight times its scale stays
// within fp16 whatever the scales are.
template <typename T, typename C, int DP, int NT>
__global__ void __launch_bounds__(kSplitThreads)
split_mma(const T* __restrict__ q, const C* __restrict__ k_cache, const C* __restrict__ v_cache,
          const int* __restrict__ table, const int* __restrict__ seq_lens,
          const float* __restrict__ k_scale, const float* __restrict__ v_scale,
          T* __restrict__ o, PagedShape sh, SplitShape sp, unsigned* err) {
  using Plan = MmaPlan<C, DP, NT>;
  using M = std::conditional_t<Plan::kQuant, __half, T>;  // operand type of the products
  constexpr bool kQuant = Plan::kQuant;
  constexpr int kS = Plan::kStages, kRow = Plan::kRow, kHeads = Plan::kHeads;
  constexpr int kKeys = Plan::kKeys, kTiles = kKeys / 16;
  constexpr int kChunks = kRow / 16;
  constexpr int kSteps = DP / 16;
  extern __shared__ __align__(128) unsigned char smem[];
  float* s_m = reinterpret_cast<float*>(smem + kSplitWarps * kS * Plan::kStage);
  float* s_l = s_m + kSplitWarps * kHeads;
  float* s_o = s_l + kSplitWarps * kHeads;
  auto* scratch = reinterpret_cast<int64_t*>(s_o + kSplitWarps * kMeetHeads * Plan::kPitch);
  const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
  const int r = lane >> 2, t = lane & 3;  // row and column pair of this lane's fragments
  const int dim = static_cast<int>(sh.lay.dim);
  const uint32_t ring = smem_u32(smem) + warp * kS * Plan::kStage;
  const int chunks_in = dim * static_cast<int>(sizeof(C)) / 16;

  pdl_launch_dependents();
  zero_empty(o, seq_lens, sh, err);
  int64_t u, end;
  UnitPlace p = find_units(seq_lens, sh, sp, scratch, &u, &end, err);
  if (u >= end) return;

  // The loader runs kS - 1 units ahead, and looks up its next unit's pages one unit before
  // that: next_row / next_scale are those of this lane's key (lane % kKeys).
  UnitPlace lp = p;
  int left = static_cast<int>(end - u);  // units that the loader has not begun
  uint32_t next_row = kNoRow, next_scale = 0;
  unsigned bad_slots = 0;
  const auto page_size = static_cast<uint32_t>(sh.lay.page_size);
  const auto page_units = static_cast<uint32_t>(sh.lay.page_stride * sizeof(C) / 16);
  auto look_up = [&]() {
    next_row = kNoRow;
    const uint32_t pos = lp.blk * Plan::kUnit + warp * kKeys + (lane & (kKeys - 1));
    if (left <= 0 || pos >= static_cast<uint32_t>(lp.n)) return;
    const uint32_t at = pos / page_size, off = pos - at * page_size;
    const int page = table[lp.b * sh.table_stride + at];
    if (page < 0 || page >= sh.lay.num_pages) {
      atomicOr(err, kErrIndex);
      next_row = kBadRow;
      return;
    }
    const uint32_t hk = static_cast<uint32_t>(lp.row) / sp.tiles;
    next_row = page * page_units + (hk * page_size + off) * chunks_in;
    next_scale = (page * static_cast<uint32_t>(sh.lay.heads) + hk) * page_size + off;
  };
  auto load = [&](int stage) {
    if (left > 0) {
      const uint32_t kd = ring + stage * Plan::kStage, vd = kd + Plan::kTile;
      const bool bad = __any_sync(kFull, next_row == kBadRow);
      bad_slots = bad ? bad_slots | (1u << stage) : bad_slots & ~(1u << stage);
#pragma unroll
      for (int i = 0; i < kKeys * kChunks / kWarp; ++i) {
        const int c = i * kWarp + lane;
        const int row = c / kChunks, ch = c % kChunks;
        const uint32_t at = __shfl_sync(kFull, next_row, row);
        const bool in = at < kBadRow && ch < chunks_in;
        const uint64_t byte = in ? static_cast<uint64_t>(at + ch) * 16 : 0;
        cp_async16(kd + tile_at<kRow>(row, ch), reinterpret_cast<const char*>(k_cache) + byte, in);
        cp_async16(vd + tile_at<kRow>(row, ch), reinterpret_cast<const char*>(v_cache) + byte, in);
      }
      if constexpr (kQuant) {  // the key scales, then the value scales
        const bool in = next_row < kBadRow;
        const uint32_t at = in ? next_scale : 0, sd = vd + Plan::kTile + lane * 4;
        if constexpr (kKeys == 32) {
          cp_async4(sd, k_scale + at, in);
          cp_async4(sd + 128, v_scale + at, in);
        } else {
          cp_async4(sd, (lane < 16 ? k_scale : v_scale) + at, in);
        }
      }
      if (--left > 0) lp.next(seq_lens, sh, sp, err);
    }
    cp_async_commit();  // an empty group where nothing is left, so that the count stays
    look_up();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < kS - 1; ++i) load(i);

  uint32_t qb[NT][kSteps][2];
  float mult[NT][2];                      // score -> log2 units, heads 2t and 2t + 1
  float acc[NT][kSteps][4];               // O^T: elements x heads
  float m[NT][2], l[NT][2], mo[NT][2];    // running maximum, sum; maximum of weight * scale
  bool fresh = true, whole_start = p.blk == 0;
  int slot = 0, stage = 0;
  for (int units = static_cast<int>(end - u); units > 0; --units) {
    if (fresh) {
      fresh = false;
      const int64_t hk = p.row / sp.tiles;
      const int first = static_cast<int>(p.row - hk * sp.tiles) * kHeads;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = first + nt * 8 + r;
        const T* qh = q + p.b * sh.q_stride + (hk * sp.group + h) * dim;
        const bool live = h < sp.group;
        if constexpr (!kQuant) {
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int d = kk * 16 + i * 8 + 2 * t;
              qb[nt][kk][i] =
                  live && d < dim ? *reinterpret_cast<const uint32_t*>(qh + d) : 0u;
            }
          }
          mult[nt][0] = mult[nt][1] = sh.scale * kLog2e;
        } else {
          // elements 4t .. 4t+3 of each 16, in the order that a word of codes has them
          uint32_t top = 0;
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
            const int d = kk * 16 + 4 * t;
            uint2 raw = make_uint2(0u, 0u);
            if (live && d < dim) raw = *reinterpret_cast<const uint2*>(qh + d);
            qb[nt][kk][0] = raw.x;
            qb[nt][kk][1] = raw.y;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const T* e = reinterpret_cast<const T*>(&qb[nt][kk][i]);
              top = max(top, __float_as_uint(to_f(e[0])) & 0x7fffffffu);
              top = max(top, __float_as_uint(to_f(e[1])) & 0x7fffffffu);
            }
          }
          top = max(top, __shfl_xor_sync(kFull, top, 1));
          top = max(top, __shfl_xor_sync(kFull, top, 2));
          // 2^-e and 2^e of the head's largest magnitude; 1 for zeros and what is not finite
          uint32_t ex = top >> 23;
          ex = ex == 0 || ex == 255 ? 127 : ex > 253 ? 253 : ex;
          const float down = __uint_as_float((254 - ex) << 23), up = __uint_as_float(ex << 23);
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const T* e = reinterpret_cast<const T*>(&qb[nt][kk][i]);
              const __half2 v = __floats2half2_rn(to_f(e[0]) * down, to_f(e[1]) * down);
              qb[nt][kk][i] = *reinterpret_cast<const uint32_t*>(&v);
            }
          }
          // `up` of heads 2t and 2t + 1 lies with the lanes of rows 2t and 2t + 1
          mult[nt][0] = __shfl_sync(kFull, up, 8 * t) * (sh.scale * kLog2e);
          mult[nt][1] = __shfl_sync(kFull, up, 8 * t + 4) * (sh.scale * kLog2e);
        }
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][kk][i] = 0.f;
        }
        m[nt][0] = m[nt][1] = mo[nt][0] = mo[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
      }
    }

    load(stage == 0 ? kS - 1 : stage - 1);
    cp_async_wait<kS - 1>();
    __syncwarp();
    const uint32_t kt = ring + stage * Plan::kStage, vt = kt + Plan::kTile;
    const int key0 = p.blk * Plan::kUnit + warp * kKeys;
    if (key0 < p.n) {  // else none of this warp's keys is left in the row
      // scores: block l / 8 of an ldmatrix is keys (l / 8) % 2 * 8 .., chunk + l / 16
      const int krow = (lane & 7) + ((lane >> 3) & 1) * 8, kch = lane >> 4;
      float c[kTiles][NT][2][4] = {};
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        if constexpr (!kQuant) {
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
            uint32_t a[4];
            ldmatrix4<false>(kt + tile_at<kRow>(krow + 16 * j, 2 * kk + kch), a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<M>(c[j][nt][kk & 1], a[0], a[1], a[2], a[3], qb[nt][kk][0], qb[nt][kk][1]);
          }
        } else {
#pragma unroll
          for (int kk = 0; kk < kSteps; kk += 2) {
            uint32_t w[4];
            ldmatrix4<false>(kt + tile_at<kRow>(krow + 16 * j, kk + kch), w);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t a0 = codes_to_half(w[2 * i]), a1 = codes_to_half(w[2 * i + 1]);
              const uint32_t a2 = codes_to_half(w[2 * i] >> 16);
              const uint32_t a3 = codes_to_half(w[2 * i + 1] >> 16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<M>(c[j][nt][i], a0, a1, a2, a3, qb[nt][kk + i][0], qb[nt][kk + i][1]);
            }
          }
        }
      }
      float ks[kTiles][2], vlog[kTiles][2];
      if constexpr (kQuant) {
        const float* sc = reinterpret_cast<const float*>(
            smem + (warp * kS + stage) * Plan::kStage + 2 * Plan::kTile);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ks[j][h] = sc[16 * j + 8 * h + r];
            vlog[j][h] = __log2f(sc[kKeys + 16 * j + 8 * h + r]);
          }
        }
      }
      const bool full = key0 + kKeys <= p.n;
      uint32_t hi[kTiles][NT][2], lo[kTiles][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[kTiles][2][2], alpha[2];  // [16 keys][key r, r + 8][head 2t, 2t + 1]
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = -INFINITY, vtop = -INFINITY;
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float s = c[j][nt][0][2 * h + i] + c[j][nt][1][2 * h + i];
              s *= kQuant ? mult[nt][i] * ks[j][h] : mult[nt][i];
              if (!full && key0 + 16 * j + 8 * h + r >= p.n) s = -INFINITY;
              w[j][h][i] = s;
              top = fmaxf(top, s);
              // past the last key the scale's place holds 0: log2 gives -inf there
              if constexpr (kQuant) vtop = fmaxf(vtop, s + vlog[j][h]);
            }
          }
#pragma unroll
          for (int off = 4; off < kWarp; off <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(kFull, top, off));
            if constexpr (kQuant) vtop = fmaxf(vtop, __shfl_xor_sync(kFull, vtop, off));
          }
          const float m_new = fmaxf(m[nt][i], top);
          const float base = m_new == -INFINITY ? 0.f : m_new;
          alpha[i] = ex2f(m[nt][i] - base);
          float sum = 0.f;
          if constexpr (kQuant) {
            const float mo_new = fmaxf(mo[nt][i], vtop);
            const float vbase = mo_new == -INFINITY ? 0.f : mo_new;
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                sum += ex2f(w[j][h][i] - (base - kWeightBits));
                w[j][h][i] = ex2f(w[j][h][i] + vlog[j][h] - (vbase - kWeightBits));
              }
            }
            l[nt][i] = fmaf(l[nt][i], alpha[i], sum);
            alpha[i] = ex2f(mo[nt][i] - vbase);
            mo[nt][i] = mo_new;
          } else {
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                w[j][h][i] = ex2f(w[j][h][i] - (base - kWeightBits));
                sum += w[j][h][i];
              }
            }
            l[nt][i] = fmaf(l[nt][i], alpha[i], sum);
          }
          m[nt][i] = m_new;
        }
        if (__any_sync(kFull, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[nt][kk][i] *= alpha[i & 1];
          }
        }
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t rest;
            hi[j][nt][h] = transpose8(split_weights<M>(w[j][h][0], w[j][h][1], &rest));
            lo[j][nt][h] = transpose8(rest);
          }
        }
      }
      // values, transposed on the way: 16-bit blocks are (keys 0-7, elements 0-7), (0-7,
      // 8-15), (8-15, 0-7), (8-15, 8-15); e4m3 blocks as for the keys, two neighbouring
      // elements of a key to a 16-bit unit
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        if constexpr (!kQuant) {
          const int vrow = (lane & 7) + (lane >> 4) * 8 + 16 * j, vch = (lane >> 3) & 1;
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
            uint32_t a[4];
            ldmatrix4<true>(vt + tile_at<kRow>(vrow, 2 * kk + vch), a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<M>(acc[nt][kk], a[0], a[1], a[2], a[3], hi[j][nt][0], hi[j][nt][1]);
              mma16816<M>(acc[nt][kk], a[0], a[1], a[2], a[3], lo[j][nt][0], lo[j][nt][1]);
            }
          }
        } else {
#pragma unroll
          for (int kk = 0; kk < kSteps; kk += 2) {
            uint32_t w[4];
            ldmatrix4<true>(vt + tile_at<kRow>(krow + 16 * j, kk + kch), w);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              // bytes: key 2t (two elements), key 2t + 1 (two) -> element by element
              const uint32_t x = __byte_perm(w[2 * i], 0, 0x3120);
              const uint32_t y = __byte_perm(w[2 * i + 1], 0, 0x3120);
              const uint32_t a0 = codes_to_half(x), a1 = codes_to_half(x >> 16);
              const uint32_t a2 = codes_to_half(y), a3 = codes_to_half(y >> 16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<M>(acc[nt][kk + i], a0, a1, a2, a3, hi[j][nt][0], hi[j][nt][1]);
                mma16816<M>(acc[nt][kk + i], a0, a1, a2, a3, lo[j][nt][0], lo[j][nt][1]);
              }
            }
          }
        }
      }
      if (bad_slots >> stage & 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = nan_f();
      }
    }
    __syncwarp();  // every lane has read this stage before it is filled again
    stage = stage + 1 == kS ? 0 : stage + 1;

    const bool row_ends = p.blk + 1 == p.blocks;
    if (row_ends || units == 1) {
      const int heads = min(kHeads, sp.group - static_cast<int>(p.row % sp.tiles) * kHeads);
      float f[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float sum = l[nt][i];
#pragma unroll
          for (int off = 4; off < kWarp; off <<= 1) sum += __shfl_xor_sync(kFull, sum, off);
          if (r == 0) {
            s_m[warp * kHeads + nt * 8 + 2 * t + i] = m[nt][i];
            s_l[warp * kHeads + nt * 8 + 2 * t + i] = sum;
          }
          // values of e4m3 rows are relative to the other maximum
          f[nt][i] = 1.f;
          if constexpr (kQuant)
            f[nt][i] = mo[nt][i] == -INFINITY ? 1.f : ex2f(mo[nt][i] - m[nt][i]);
        }
      }
#pragma unroll
      for (int h0 = 0; h0 < kHeads; h0 += kMeetHeads) {
        if (h0 >= heads) break;
        const int nt = h0 / 8, at_t = t - (h0 % 8) / 2;  // this round's heads: nt, t of 0 .. 1
        if (at_t == 0 || at_t == 1) {
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
            const int d0 = kk * 16 + (kQuant ? 2 * r : r), d1 = d0 + (kQuant ? 1 : 8);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float* at = s_o + (warp * kMeetHeads + 2 * at_t + i) * Plan::kPitch;
              at[d0] = acc[nt][kk][i] * f[nt][i];
              at[d1] = acc[nt][kk][2 + i] * f[nt][i];
            }
          }
        }
        __syncthreads();
        write_segment(s_m, s_l, s_o, h0, kMeetHeads, p, whole_start && row_ends, slot, o, sh, sp);
        __syncthreads();
      }
      fresh = true;
      whole_start = true;
      slot = 1;
    }
    p.next(seq_lens, sh, sp, err);
  }
  cp_async_wait<0>();
}

// ------------------------------------------------------------------ launch

struct PagedCall {
  const void *q, *k_cache, *v_cache;
  const int *table, *seq_lens;
  const float *k_scale, *v_scale;
  void* o;
  PagedShape sh;
  unsigned* err;
  cudaStream_t s;
};

// The widest grid: what bounds a call's partials, two per CTA of tile_heads x pitch floats.
constexpr int64_t kMaxCtas = 1024;

int64_t partial_floats(int tile_heads, int pitch) {
  return int64_t{2} * tile_heads * pitch;
}

size_t bases_bytes(int64_t batch) {
  return static_cast<size_t>(cdiv((batch + 1) * static_cast<int64_t>(sizeof(int64_t)), 16) * 16);
}

// Units of a call if every sequence were as long as its table allows.
int64_t units_bound(int64_t batch, int64_t rows, int64_t max_len, int unit) {
  const int64_t per = cdiv(max_len, unit) * rows;
  return per == 0 ? 0 : batch > INT64_MAX / 4096 / per ? INT64_MAX / 4096 : batch * per;
}

// Grid of the first kernel: one wave, no more CTAs than units.
int64_t split_ctas(int64_t units, int64_t resident) {
  return std::max<int64_t>(1, std::min({units, resident, kMaxCtas}));
}

template <typename T>
int launch_join(const PagedCall& c, const SplitShape& sp, int64_t ctas) {
  const int64_t max_len = c.sh.max_pages * c.sh.lay.page_size;
  if (max_len <= int64_t{1} << sp.unit_log) return KPB_OK;  // no row has a second unit to share
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(c.sh.batch * sp.rows));
  cfg.blockDim = dim3(kJoinWarps * kWarp);
  cfg.stream = c.s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  KPB_CUDA(cudaLaunchKernelEx(&cfg, join_rows<T>, c.seq_lens, static_cast<T*>(c.o), c.sh, sp, ctas,
                              c.err));
  return KPB_OK;
}

SplitShape split_shape(const PagedCall& c, int tile_heads, int pitch, int unit, void* ws) {
  SplitShape sp;
  sp.group = static_cast<int>(c.sh.q_heads / c.sh.lay.heads);
  sp.tile_heads = tile_heads;
  sp.tiles = static_cast<int>(cdiv(sp.group, tile_heads));
  sp.rows = c.sh.lay.heads * sp.tiles;
  sp.pitch = pitch;
  for (sp.unit_log = 0; 1 << sp.unit_log < unit; ++sp.unit_log) {
  }
  sp.bases = static_cast<int64_t*>(ws);
  sp.partials = reinterpret_cast<float*>(static_cast<char*>(ws) + bases_bytes(c.sh.batch));
  return sp;
}

template <typename T, typename C, int E, int HG>
int launch_simt(const PagedCall& c, void* ws) {
  const SplitShape sp = split_shape(c, HG, E * kWarp + 4, kSimtUnit, ws);
  auto* kernel = split_simt<T, C, E, HG>;
  int occ = 0;
  if (int rc = occupancy_blocks(reinterpret_cast<const void*>(kernel), kSplitThreads, 0, &occ))
    return rc;
  const int64_t units = units_bound(c.sh.batch, sp.rows, c.sh.max_pages * c.sh.lay.page_size, kSimtUnit);
  const int64_t ctas = split_ctas(units, int64_t{occ} * sm_count());
  kernel<<<static_cast<unsigned>(ctas), kSplitThreads, 0, c.s>>>(
      static_cast<const T*>(c.q), static_cast<const C*>(c.k_cache),
      static_cast<const C*>(c.v_cache), c.table, c.seq_lens, c.k_scale, c.v_scale,
      static_cast<T*>(c.o), c.sh, sp, c.err);
  KPB_LAUNCHED("paged_attention split");
  return launch_join<T>(c, sp, ctas);
}

// Heads per tile: the smallest of 1, 2, 4, 8 that holds the group, 8 for larger ones.
template <typename T, typename C, int E>
int dispatch_simt_heads(const PagedCall& c, void* ws) {
  const int64_t group = c.sh.q_heads / c.sh.lay.heads;
  if (group <= 1) return launch_simt<T, C, E, 1>(c, ws);
  if (group <= 2) return launch_simt<T, C, E, 2>(c, ws);
  if (group <= 4) return launch_simt<T, C, E, 4>(c, ws);
  return launch_simt<T, C, E, 8>(c, ws);
}

template <typename T, typename C>
int dispatch_simt(const PagedCall& c, void* ws) {
  if (c.sh.lay.dim <= 64) return dispatch_simt_heads<T, C, 2>(c, ws);
  if (c.sh.lay.dim <= 128) return dispatch_simt_heads<T, C, 4>(c, ws);
  return dispatch_simt_heads<T, C, 8>(c, ws);
}

template <typename T, typename C, int DP, int NT>
int launch_mma(const PagedCall& c, void* ws) {
  using Plan = MmaPlan<C, DP, NT>;
  const SplitShape sp = split_shape(c, Plan::kHeads, Plan::kPitch, Plan::kUnit, ws);
  auto* kernel = split_mma<T, C, DP, NT>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  if (int rc = ensure_dyn_smem(fn, Plan::kSmem)) return rc;
  int occ = 0;
  if (int rc = occupancy_blocks(fn, kSplitThreads, Plan::kSmem, &occ)) return rc;
  const int64_t units = units_bound(c.sh.batch, sp.rows, c.sh.max_pages * c.sh.lay.page_size, Plan::kUnit);
  const int64_t ctas = split_ctas(units, int64_t{occ} * sm_count());
  kernel<<<static_cast<unsigned>(ctas), kSplitThreads, Plan::kSmem, c.s>>>(
      static_cast<const T*>(c.q), static_cast<const C*>(c.k_cache),
      static_cast<const C*>(c.v_cache), c.table, c.seq_lens, c.k_scale, c.v_scale,
      static_cast<T*>(c.o), c.sh, sp, c.err);
  KPB_LAUNCHED("paged_attention split");
  return launch_join<T>(c, sp, ctas);
}

// Sixteen heads to a tile where the group has more than eight, so that its keys are read
// once; at D > 128 their sums would not fit the registers.
template <typename T, typename C>
int dispatch_mma(const PagedCall& c, void* ws) {
  const bool wide = c.sh.q_heads / c.sh.lay.heads > 8;
  if (c.sh.lay.dim <= 64)
    return wide ? launch_mma<T, C, 64, 2>(c, ws) : launch_mma<T, C, 64, 1>(c, ws);
  if (c.sh.lay.dim <= 128)
    return wide ? launch_mma<T, C, 128, 2>(c, ws) : launch_mma<T, C, 128, 1>(c, ws);
  return launch_mma<T, C, 256, 1>(c, ws);
}

// Rows of the cache whole 16-byte chunks on 16-byte boundaries (cp.async), q's rows on
// 8-byte ones; the cache's 16-byte units counted in 32 bits (64 GB, of 180 on the card).
template <typename C>
bool mma_takes(const PagedCall& c) {
  const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  return c.sh.lay.dim * sizeof(C) % 16 == 0 && c.sh.lay.dim % 8 == 0 &&
         (at(c.k_cache) | at(c.v_cache)) % 16 == 0 &&
         (c.sh.lay.num_pages < 2 || c.sh.lay.page_stride * sizeof(C) % 16 == 0) &&
         c.sh.lay.num_pages * c.sh.lay.page_stride * static_cast<int64_t>(sizeof(C)) / 16 < kBadRow &&
         at(c.q) % 8 == 0 && (c.sh.batch < 2 || c.sh.q_stride % 4 == 0);
}

template <typename T, typename C>
int launch(int variant, const PagedCall& c, void* ws) {
  if (variant == 0) {
    paged_cta_head<T, C><<<static_cast<unsigned>(c.sh.batch * c.sh.q_heads), 128, 0, c.s>>>(
        static_cast<const T*>(c.q), static_cast<const C*>(c.k_cache),
        static_cast<const C*>(c.v_cache), c.table, c.seq_lens, c.k_scale, c.v_scale,
        static_cast<T*>(c.o), c.sh, c.err);
    KPB_LAUNCHED("paged_attention variant 0");
    return KPB_OK;
  }
  if constexpr (sizeof(T) == 2) {
    if (mma_takes<C>(c)) return dispatch_mma<T, C>(c, ws);
  }
  return dispatch_simt<T, C>(c, ws);
}

}  // namespace

size_t paged_attention_workspace_bytes(int variant, int64_t batch, int64_t q_heads,
                                       int64_t k_heads, int64_t dim, int64_t max_len) {
  if (variant == 0) return 0;
  // the widest tile and pitch that any of the ways takes for this call, and as many CTAs as
  // there can be units (a tile holds one head at least)
  const int pitch = static_cast<int>(dim <= 64 ? 64 : dim <= 128 ? 128 : 256) + 4;
  const int heads = q_heads / k_heads > 8 && dim <= 128 ? 16 : 8;
  const int64_t ctas = split_ctas(units_bound(batch, q_heads, max_len, kSimtUnit), kMaxCtas);
  return bases_bytes(batch) +
         static_cast<size_t>(ctas * partial_floats(heads, pitch)) * sizeof(float);
}

int paged_attention(int variant, int dtype, int cache_dtype, const void* q, const void* k_cache,
                    const void* v_cache, const int* table, const int* seq_lens,
                    const float* k_scale, const float* v_scale, void* o, int64_t batch,
                    int64_t q_heads, int64_t max_pages, int64_t q_stride, int64_t table_stride,
                    float scale, const KvLayout& lay, void* ws, size_t ws_bytes, unsigned* err,
                    cudaStream_t s) {
  const PagedCall c{q,       k_cache, v_cache, table, seq_lens, k_scale, v_scale, o,
                    PagedShape{batch, q_heads, max_pages, q_stride, table_stride, scale, lay},
                    err,     s};
  const bool e4m3 = cache_dtype == KPB_E4M3;
  switch (dtype) {
    case KPB_F32:
      return e4m3 ? launch<float, uint8_t>(variant, c, ws) : launch<float, float>(variant, c, ws);
    case KPB_F16:
      return e4m3 ? launch<__half, uint8_t>(variant, c, ws) : launch<__half, __half>(variant, c, ws);
    default:
      return e4m3 ? launch<__nv_bfloat16, uint8_t>(variant, c, ws)
                  : launch<__nv_bfloat16, __nv_bfloat16>(variant, c, ws);
  }
}

}  // namespace kpb
