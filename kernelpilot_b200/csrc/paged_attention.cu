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
//   variant 1  the keys of all sequences split evenly over the warps of one wave of CTAs,
//              whatever the lengths are. A unit of work is 16 or 32 keys of one row, a row
//              being a (sequence, key head, tile of its query heads); every worker takes as
//              many units as any other, give or take one, found from the lengths on the
//              device, so one captured call serves any lengths. A row that lies with one
//              warp is finished there; of one that several share each leaves a partial
//              (maximum, sum, weighted values), joined in order by a second kernel (a
//              programmatic dependent). Each warp streams its own keys and values and no
//              barrier stands in its way: with the four warps of a CTA on one row instead,
//              meeting in shared memory at each row's end, the calls below took 13.6 us for
//              the one sequence and 113 for e4m3 (10.7 and 103 with warps at that step; the
//              bf16 batch 173 and 175). Two ways to the products:
//                split_mma   fp16 / bf16 q, or fp32 q on an e4m3 cache up to D = 128, rows
//                            a multiple of 16 bytes on 16-byte boundaries: cp.async
//                            into a swizzled ring per warp, mma.sync (a key head's
//                            1 to 16 query heads fill 8-wide fragments; of a 128-row
//                            tcgen05 tile they would fill a few rows, and the tensor
//                            pipe is 16 to 28% busy as it is)
//                split_simt  everything else (fp32 caches, odd head dims, odd bases)
//
// What bounds it: the keys' and values' bytes; for e4m3, with half the bytes a value, their
// conversion to fp16 and the warps' latency as much. Measured on B200 (6464 GB/s copy), head
// dim 128, 8 key heads, ragged lengths:
//   64 sequences up to 8192 keys, bf16, 32 query heads    174 us (1065 MB; 165 at that rate)
//   32 sequences up to 16384 keys, e4m3, 64 query heads   103 us (549 MB; 85)
//   64 sequences up to 4096 keys, fp32, 32 query heads    184 us (1066 MB; 165)
//   2 sequences up to 32768 keys, fp16, 32 heads of 64     77 us (434 MB; 67)
//   one sequence of 1037 keys, bf16, 32 query heads       11.0 us, 3 of them the join's launch
// variant 0 takes 4764, 9193, -, 12317 and 274 us on the same calls.
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

// How rows and units are laid out: a unit is a power of two of keys of a row; rows of a
// sequence are (key head, tile of `tile_heads` query heads), tiles innermost; a partial has
// tile_heads x pitch floats: pitch - 4 weighted values, then maximum and sum.
struct SplitShape {
  int64_t rows;      // rows per sequence
  int tiles;         // tiles of query heads per key head
  int group;         // query heads per key head
  int tile_heads;
  int pitch;
  int unit_log;      // log2 of the keys per unit
  int deal_log;      // log2 of the keys dealt out at a time: a unit, or a whole short row
  int page_log;      // log2 of the page size, -1 where it is no power of two
  int2* shared;      // workspace: [sequence][row], (first partial, partials) where workers share it
  float* partials;   // workspace: [worker][2][tile_heads][pitch]
};

// Units of a row of n keys.
__device__ __forceinline__ int units_of(int64_t n, const SplitShape& sp) {
  return static_cast<int>((n + (1 << sp.unit_log) - 1) >> sp.unit_log);
}

// a / b for a >= 0, b > 0: 64-bit division takes the better part of a microsecond, and the
// operands nearly always fit 32 bits.
__device__ __forceinline__ int64_t div_fast(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

// How `total` units are dealt out: `each` to a worker and one more to the first `extra`.
struct Deal {
  int64_t each, extra;

  __device__ __forceinline__ Deal(int64_t total, int64_t workers)
      : each(div_fast(total, workers)), extra(total - each * workers) {}
  __device__ __forceinline__ int64_t first(int64_t worker) const {
    return worker * each + min(worker, extra);
  }
  __device__ __forceinline__ int64_t worker_of(int64_t unit) const {
    const int64_t more = extra * (each + 1);
    return unit < more ? div_fast(unit, each + 1) : extra + div_fast(unit - more, each);
  }
};

// Shares that a row of n keys is dealt out in.
__device__ __forceinline__ int shares_of(int64_t n, const SplitShape& sp) {
  return static_cast<int>((n + (1 << sp.deal_log) - 1) >> sp.deal_log);
}

// Workers of a grid: its warps, but two units to a worker at least once there are 64 workers
// (the second unit's loads run beside the first's; a worker less is a partial less to join).
// Never more workers than shares, so that every worker of a shared row has a part of it.
constexpr int kMinUnits = 2;

__device__ __forceinline__ int64_t workers_of(int64_t ctas, int64_t total, const SplitShape& sp) {
  const int64_t most =
      sp.deal_log > sp.unit_log ? total : max(total / kMinUnits, min(total, int64_t{64}));
  return min(ctas * kSplitWarps, most);
}

// A place in the list of units: sequence, row, block of keys. The lengths are read several
// times over; should another stream change them under a call, its results mean nothing, but
// every loop here still ends at the last sequence and no partial past the workspace is read.
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

// What find_units needs of shared memory; total stays there.
struct FindScratch {
  int64_t warp_sum[kSplitWarps], upto[kSplitThreads], total;
};

// This warp's worker number, its count of units and the place of the first. Every thread
// calls it: thread i adds up the units of the i-th run of sequences, a scan gives each run
// its first unit, and each warp looks its own unit up among the runs. Workers are dealt out
// over the CTAs first, so that few units spread over all SMs.
__device__ __forceinline__ UnitPlace find_units(const int* __restrict__ seq_lens,
                                                const PagedShape& sh, const SplitShape& sp,
                                                FindScratch* scratch, int64_t* worker, int* count,
                                                unsigned* err) {
  const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
  const int64_t per = (sh.batch + kSplitThreads - 1) / kSplitThreads;
  const int64_t b0 = min(sh.batch, threadIdx.x * per), b1 = min(sh.batch, b0 + per);
  int64_t mine = 0;
  for (int64_t b = b0; b < b1; ++b)
    mine += shares_of(keys_of(seq_lens, b, sh, err), sp) * sp.rows;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < kWarp; o <<= 1) {
    const int64_t v = __shfl_up_sync(kFull, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == kWarp - 1) scratch->warp_sum[warp] = upto;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kSplitWarps; ++w) {
    if (w < warp) upto += scratch->warp_sum[w];
    total += scratch->warp_sum[w];
  }
  scratch->upto[threadIdx.x] = upto;
  if (threadIdx.x == 0) scratch->total = total;
  __syncthreads();
  const int64_t workers = workers_of(gridDim.x, total, sp);
  *worker = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;
  UnitPlace p = {};
  *count = 0;
  if (*worker >= workers) return p;
  const Deal deal(total, workers);
  const int64_t begin = deal.first(*worker);
  *count = static_cast<int>(deal.first(*worker + 1) - begin);
  // the run that holds `begin`: as many runs end at or before it
  int before = 0;
#pragma unroll
  for (int i = 0; i < kSplitThreads / kWarp; ++i)
    before += __popc(__ballot_sync(kFull, scratch->upto[i * kWarp + lane] <= begin));
  int64_t base = before == 0 ? 0 : scratch->upto[before - 1];
  int shares = 0;
  for (p.b = before * per; p.b < sh.batch; ++p.b) {
    p.n = static_cast<int>(keys_of(seq_lens, p.b, sh, err));
    shares = shares_of(p.n, sp);
    if (begin < base + shares * sp.rows) break;
    base += shares * sp.rows;
  }
  if (p.b >= sh.batch) {  // only where the lengths change under the call
    *count = 0;
    return p;
  }
  p.blocks = units_of(p.n, sp);
  p.row = div_fast(begin - base, shares);
  p.blk = static_cast<int>(begin - base - p.row * shares);  // 0 where whole rows are dealt out
  if (sp.deal_log > sp.unit_log) {  // the units of the worker's rows, sequence by sequence
    int left = *count, units = 0;
    int64_t row = p.row;
    for (int64_t b = p.b; left > 0 && b < sh.batch; ++b, row = 0) {
      const int blocks = units_of(keys_of(seq_lens, b, sh, err), sp);
      if (blocks == 0) continue;
      const int rows = static_cast<int>(min(static_cast<int64_t>(left), sp.rows - row));
      units += rows * blocks;
      left -= rows;
    }
    *count = units;
  }
  return p;
}

// Zeros for the sequences without keys, strided over the CTAs; no worker shares their rows.
template <typename T>
__device__ __forceinline__ void zero_empty(T* __restrict__ o, const int* __restrict__ seq_lens,
                                           const PagedShape& sh, const SplitShape& sp,
                                           unsigned* err) {
  const int64_t row = sh.q_heads * sh.lay.dim;
  for (int64_t b = blockIdx.x; b < sh.batch; b += gridDim.x) {
    if (keys_of(seq_lens, b, sh, err) != 0) continue;
    for (int64_t i = threadIdx.x; i < row; i += kSplitThreads) o[b * row + i] = from_f<T>(0.f);
    for (int64_t i = threadIdx.x; i < sp.rows; i += kSplitThreads)
      sp.shared[b * sp.rows + i] = make_int2(0, 0);
  }
}

// Partial `slot` (0: of a row that began before this worker, 1: of one that did not) of a
// worker, head h of the tile.
__device__ __forceinline__ float* partial_at(const SplitShape& sp, int64_t worker, int slot,
                                             int h) {
  return sp.partials + ((worker * 2 + slot) * sp.tile_heads + h) * sp.pitch;
}

// Says for the row of place p, whose first unit this worker had, which partials it is in:
// none if it is `whole`, else this worker's `slot` and slot 0 of the workers after it up to
// the one with the row's last unit. `left`: this worker's units from p on.
__device__ __forceinline__ void note_shared(const UnitPlace& p, bool whole, int64_t worker,
                                            int slot, int left, const FindScratch* scratch,
                                            const SplitShape& sp) {
  int2 note = make_int2(0, 0);
  if (!whole) {
    const int64_t workers = workers_of(gridDim.x, scratch->total, sp);
    const Deal deal(scratch->total, workers);
    const int64_t last = deal.first(worker + 1) - left + (p.blocks - 1 - p.blk);
    note = make_int2(static_cast<int>(worker * 2 + slot),
                     static_cast<int>(min(deal.worker_of(last), workers - 1) - worker) + 1);
  }
  sp.shared[p.b * sp.rows + p.row] = note;
}

// The partials of a (sequence, query head) whose row several workers share, joined by
// 2^share_log of a CTA's warps: each takes every so manieth partial, lanes strided over the
// values, as out = sum_c f_c O_c / sum_c f_c l_c, f_c = 2^(m_c - max m) carried along as a
// running maximum; then the warps in order.
constexpr int kJoinWarps = 16;

template <typename T, int E>
__global__ void __launch_bounds__(kJoinWarps * kWarp)
join_rows(T* __restrict__ o, int heads, int dim, SplitShape sp, int workers, int share_log) {
  __shared__ float s_m[kJoinWarps], s_l[kJoinWarps], s_o[kJoinWarps][E * kWarp];
  const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
  constexpr int kAhead = E == 8 ? 4 : 8;
  const int share = 1 << share_log, part = warp & (share - 1), first_warp = warp - part;
  // head `at` of all sequences' heads: group at / sp.group of all key heads
  const int64_t head = static_cast<int64_t>(blockIdx.x) * (kJoinWarps >> share_log) +
                       (warp >> share_log);
  const int at = static_cast<int>(head);
  const bool live = head < heads;
  const int hk = live ? at / sp.group : 0, g = live ? at - hk * sp.group : 0;
  const int tile = g / sp.tile_heads;
  pdl_wait_primary();
  const int2 note = live ? sp.shared[static_cast<int64_t>(hk) * sp.tiles + tile] : make_int2(0, 0);
  const int count = note_is_sound(note.x, note.y, workers) ? note.y : 0;
  float m = -INFINITY, l = 0.f, acc[E] = {};
  if (count > 1) {
    const int h = g - tile * sp.tile_heads;
    const float* p0 = partial_at(sp, note.x >> 1, note.x & 1, h);
    const float* rest = partial_at(sp, note.x >> 1, 0, h);
    const int64_t step = static_cast<int64_t>(2) * sp.tile_heads * sp.pitch;
    // kAhead partials are loaded before the first is used, the last few under a guard
    for (int c0 = part; c0 < count; c0 += kAhead * share) {
      float v[kAhead][E], pm[kAhead], pl[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int c = c0 + i * share;
        const float* p = c == 0 ? p0 : rest + c * step;
        pm[i] = c < count ? p[E * kWarp] : -INFINITY;
        pl[i] = c < count ? p[E * kWarp + 1] : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) v[i][e] = c < count ? p[lane + e * kWarp] : 0.f;
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) top = fmaxf(top, pm[i]);
      const float to = top == -INFINITY ? 0.f : top, f = ex2f(m - to);
      l *= f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float pf = ex2f(pm[i] - to);
        l = fmaf(pl[i], pf, l);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(v[i][e], pf, acc[e]);
      }
      m = top;
    }
  }
  if (share > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane + e * kWarp] = acc[e];
    if (lane == 0) {
      s_m[warp] = m;
      s_l[warp] = l;
    }
    __syncthreads();
    if (part != 0) return;
    for (int w = first_warp + 1; w < first_warp + share; ++w) {
      const float top = fmaxf(m, s_m[w]), to = top == -INFINITY ? 0.f : top;
      const float f = ex2f(m - to), pf = ex2f(s_m[w] - to);
      l = fmaf(l, f, s_l[w] * pf);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(acc[e], f, s_o[w][lane + e * kWarp] * pf);
      m = top;
    }
  }
  if (count < 2) return;
  T* out = o + head * dim;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = lane + e * kWarp;
    if (i < dim) out[i] = from_f<T>(acc[e] / l);
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

constexpr int kSimtUnit = 16;
constexpr int kSimtKeys = 4;  // keys that a warp takes at a time

// Stages of the ring of 4 keys and values per thread: up to 64 KB a CTA.
constexpr int simt_stages(int E) { return E == 8 ? 2 : E == 4 ? 3 : 4; }
constexpr int simt_ring_bytes(int E) {
  return simt_stages(E) * kSimtKeys * 2 * E * 4 * kSplitThreads;
}
constexpr int simt_vector(int E) { return E == 2 ? 2 : 4; }

// A lane holds E of a row's elements; a warp takes 4 keys at a time and HG query heads:
// 4 * HG products, summed over the lanes by halving, so that each lane ends with the score
// of one (key, head). kRing (fp32 rows in whole vectors): elements in vectors of 8 or 16
// bytes, each thread's own through its own slots of a shared-memory ring, groups of 4 keys
// simt_stages - 1 ahead. Else: elements strided over the lanes, read where they are used.
template <typename T, typename C, int E, int HG, bool kRing>
__global__ void __launch_bounds__(kSplitThreads)
split_simt(const T* __restrict__ q, const C* __restrict__ k_cache, const C* __restrict__ v_cache,
           const int* __restrict__ table, const int* __restrict__ seq_lens,
           const float* __restrict__ k_scale, const float* __restrict__ v_scale,
           T* __restrict__ o, PagedShape sh, SplitShape sp, unsigned* err) {
  constexpr int kKeys = kSimtKeys;
  constexpr int kSums = kKeys * HG;
  constexpr int kLog = kSums == 32 ? 5 : kSums == 16 ? 4 : kSums == 8 ? 3 : 2;
  constexpr int kSpread = 5 - kLog;  // 2^kSpread neighbouring lanes hold the same sum
  constexpr bool kQuant = std::is_same_v<C, uint8_t>;
  __shared__ FindScratch scratch;
  const int lane = threadIdx.x & (kWarp - 1);
  const int dim = static_cast<int>(sh.lay.dim);
  pdl_launch_dependents();
  int64_t worker;
  int count;
  UnitPlace p = find_units(seq_lens, sh, sp, &scratch, &worker, &count, err);
  const int my_key = (lane >> kSpread) / HG;
  constexpr int VE = kRing ? simt_vector(E) : 1, kVectors = E / VE, kS = simt_stages(E);
  const auto element = [&](int e) { return (e / VE * kWarp + lane) * VE + e % VE; };

  // the ring's loader: the unit, group of keys and rows (lane j: key j of the unit) that it
  // loads next, and which of the units in flight hold a bad page
  extern __shared__ __align__(16) float ring[];
  UnitPlace lp = p;
  int left = kRing ? count : 0, group = 0;
  int64_t next_row = -1, unused = 0;
  unsigned bad_units = 0, load_unit = 0, unit = 0;
  const auto slot_of = [&](int stage, int key, int which, int v) {
    return ((((stage * kKeys + key) * 2 + which) * kVectors + v) * kSplitThreads +
            static_cast<int>(threadIdx.x)) * VE;
  };
  const auto look_up = [&]() {
    next_row = -1;
    if (left > 0 && lane < kSimtUnit)
      next_row = key_row(table, lp.b, lp.blk * kSimtUnit + lane, lp.n,
                         static_cast<uint32_t>(lp.row) / sp.tiles, sh, &unused, err);
  };
  const auto load = [&](int stage) {
    if (left > 0) {
      if (group == 0) {
        const unsigned bit = 1u << (load_unit & 31);
        bad_units = __any_sync(kFull, next_row == -2) ? bad_units | bit : bad_units & ~bit;
      }
#pragma unroll
      for (int k = 0; k < kKeys; ++k) {
        const int64_t row = __shfl_sync(kFull, next_row, group * kKeys + k);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
          const int i = element(v * VE);
          const bool in = row >= 0 && i < dim;
          const int64_t at = in ? row + i : 0;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const auto* src = reinterpret_cast<const char*>((w == 0 ? k_cache : v_cache) + at);
            const uint32_t dst = smem_u32(ring + slot_of(stage, k, w, v));
            if constexpr (VE == 4) cp_async16(dst, src, in);
            else cp_async8(dst, src, in);
          }
        }
      }
      if (++group * kKeys >= min(kSimtUnit, lp.n - lp.blk * kSimtUnit)) {
        group = 0;
        ++load_unit;
        if (--left > 0) lp.next(seq_lens, sh, sp, err);
        if (lp.b >= sh.batch) left = 0;
        look_up();
      }
    }
    cp_async_commit();  // an empty group where nothing is left, so that the count stays
  };
  int stage = 0;
  if constexpr (kRing) {
    look_up();
#pragma unroll
    for (int i = 0; i < kS - 1; ++i) load(i);
  }

  float qr[HG][E], acc[HG][E], m = -INFINITY, l = 0.f;
  bool fresh = true, whole_start = p.blk == 0;
  int slot = 0;
  for (; count > 0 && p.b < sh.batch; --count) {
    const int64_t hk = static_cast<uint32_t>(p.row) / sp.tiles;
    const int first = static_cast<int>(p.row - hk * sp.tiles) * HG;
    if (fresh) {
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const T* qh = q + p.b * sh.q_stride + (hk * sp.group + first + h) * dim;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = element(e);
          qr[h][e] = i < dim && first + h < sp.group ? to_f(qh[i]) * (sh.scale * kLog2e) : 0.f;
          acc[h][e] = 0.f;
        }
      }
      m = -INFINITY;
      l = 0.f;
      fresh = false;
    }
    const int key0 = p.blk * kSimtUnit;
    int64_t my_scale = 0;
    int64_t my_row = -1;
    if constexpr (!kRing) {
      if (lane < kSimtUnit) my_row = key_row(table, p.b, key0 + lane, p.n, hk, sh, &my_scale, err);
    }
    if (kRing ? bad_units >> (unit++ & 31) & 1 : __any_sync(kFull, my_row == -2)) l = nan_f();
    float ks = 1.f, vs = 1.f;
    if constexpr (kQuant) {
      if (my_row >= 0) {
        ks = k_scale[my_scale];
        vs = v_scale[my_scale];
      }
    }
#pragma unroll 1
    for (int j = 0; j < kSimtUnit && key0 + j < p.n; j += kKeys) {
      float kv[kKeys][E], vv[kKeys][E];
      if constexpr (kRing) {
        load(stage == 0 ? kS - 1 : stage - 1);
        cp_async_wait<kS - 1>();
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {
#pragma unroll
          for (int v = 0; v < kVectors; ++v) {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              kv[k][v * VE + e] = ring[slot_of(stage, k, 0, v) + e];
              vv[k][v * VE + e] = ring[slot_of(stage, k, 1, v) + e];
            }
          }
        }
        stage = stage + 1 == kS ? 0 : stage + 1;
      } else {
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {
          const int64_t row = __shfl_sync(kFull, my_row, j + k);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const int i = element(e);
            const bool in = i < dim && row >= 0;
            kv[k][e] = in ? cache_value(k_cache + row, i, 1.f) : 0.f;
            vv[k][e] = in ? cache_value(v_cache + row, i, 1.f) : 0.f;
          }
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
      if (key0 + j + my_key >= p.n) score = -INFINITY;
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
    if (row_ends || count == 1) {
      float sum = l;
#pragma unroll
      for (int off = HG << kSpread; off < kWarp; off <<= 1)
        sum += __shfl_xor_sync(kFull, sum, off);
      const bool whole = whole_start && row_ends;
      if (whole_start && lane == 0) note_shared(p, whole, worker, slot, count, &scratch, sp);
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const float hs = __shfl_sync(kFull, sum, h << kSpread);
        const float hm = __shfl_sync(kFull, m, h << kSpread);
        if (first + h >= sp.group) break;
        T* out = o + (p.b * sh.q_heads + hk * sp.group + first + h) * dim;
        float* part = partial_at(sp, worker, slot, h);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = element(e);
          if (!whole) part[i] = acc[h][e];
          else if (i < dim) out[i] = from_f<T>(acc[h][e] / hs);
        }
        if (!whole && lane == 0) {
          part[E * kWarp] = hm;
          part[E * kWarp + 1] = hs;
        }
      }
      fresh = true;
      whole_start = true;
      slot = 1;
    }
    p.next(seq_lens, sh, sp, err);
  }
  if constexpr (kRing) cp_async_wait<0>();
  zero_empty(o, seq_lens, sh, sp, err);
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

// fp16 weights are held times 2^14 (the maximum's weight is 16384): they keep their full
// fraction down to 2^-28 of the largest and something down to 2^-38. bf16 has fp32's range, and
// its weights are held as they are: 2^14 would bring sums of values from 2^114 on to infinity.
template <typename M>
constexpr float kWeightBits = std::is_same_v<M, __half> ? 14.f : 0.f;
template <typename M>
constexpr float kWeightUnit = std::is_same_v<M, __half> ? 0x1p-14f : 1.f;

// The smallest fp16 number.
constexpr float kHalfTiny = 0x1p-24f;

// Weights w >= 0 as a pair of M (x in the low half), and as *rest what that leaves. Where
// the values may hold infinities (kCut: not e4m3 codes) the pair is cut towards zero and the
// rest is never 0 beside a weight that is not (fp16: that kHalfTiny is not above): an infinite
// value times the two is then an infinity, not infinity * 0 or the difference of two.
template <typename M, bool kCut>
__device__ __forceinline__ uint32_t split_weights(float x, float y, uint32_t* rest) {
  constexpr float kTiny = std::is_same_v<M, __half> ? kHalfTiny : 0x1p-120f;
  uint32_t hi;
  float2 f;
  if constexpr (std::is_same_v<M, __half>) {
    if constexpr (kCut) asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
    f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  } else {
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
    f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&hi));
  }
  float rx = x - f.x, ry = y - f.y;
  if constexpr (kCut) {
    rx = fmaxf(rx, fminf(x, kTiny));
    ry = fmaxf(ry, fminf(y, kTiny));
  }
  if constexpr (std::is_same_v<M, __half>) {
    const __half2 v = __floats2half2_rn(rx, ry);
    *rest = *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(rx, ry);
    *rest = *reinterpret_cast<const uint32_t*>(&v);
  }
  return hi;
}

// Whether a tile of `bytes` bytes of fp16 holds an infinity (same answer in every lane).
__device__ __forceinline__ bool tile_has_inf(const unsigned char* tile, int bytes) {
  __half2 top = __half2half2(__ushort_as_half(0));  // NaNs stay out of the maximum
  for (int i = (threadIdx.x & (kWarp - 1)) * 16; i < bytes; i += kWarp * 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(tile + i);
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __hmax2(top, __habs2(h[e]));
  }
  return __any_sync(kFull, __hisinf(__low2half(top)) != 0 || __hisinf(__high2half(top)) != 0);
}

// Queries of e4m3 products are held with the head's largest element at 2^14 to 2^15, the top
// of fp16's range; the products' sums (2^15 x 448 x 256 at most) have room for it in fp32.
constexpr uint32_t kQueryBits = 14;

// Four e4m3 codes as two pairs of fp16, exactly.
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t* lo, uint32_t* hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(*lo), "=r"(*hi) : "r"(w));
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

// tile_at(row0 + lr, ch) for a constant row0 and lr < the rows of a turn (which divide 8, or
// are 8): the exchange splits into a constant part and one that stays.
template <int kRow>
__device__ __forceinline__ uint32_t tile_turn(int row0, int lr, int ch) {
  const uint32_t mine = static_cast<uint32_t>(
      lr * kRow + ((ch ^ (kRow >= 128 ? lr : lr >> 1 & 3)) << 4));
  return row0 * kRow + (mine ^ static_cast<uint32_t>(kRow >= 128 ? (row0 & 7) << 4 : 0));
}

// Whether row `row` of a tile of e4m3 codes is all zeros (of either sign).
template <int kRow>
__device__ __forceinline__ bool row_is_zero(const unsigned char* tile, int row) {
#pragma unroll 1
  for (int ch = 0; ch < kRow / 16; ++ch) {
    const uint4 v = *reinterpret_cast<const uint4*>(tile + tile_at<kRow>(row, ch));
    if (((v.x | v.y | v.z | v.w) & 0x7f7f7f7fu) != 0) return false;
  }
  return true;
}

// Shared memory of one CTA: kStages x (keys, values, scales) per warp. A warp takes 32 keys
// at a time where a row is 128 bytes at most, else 16. As many stages as let three CTAs
// share an SM, two at least and four at most; where two do not fit, two CTAs or one.
template <typename C, int DP, int NT>
struct MmaPlan {
  static constexpr bool kQuant = std::is_same_v<C, uint8_t>;
  static constexpr int kRow = DP * static_cast<int>(sizeof(C));
  static constexpr int kKeys = kRow <= 128 && DP * NT <= 128 ? 32 : 16;
  static constexpr int kTile = kKeys * kRow;
  static constexpr int kStage = 2 * kTile + (kQuant ? 2 * kKeys * 4 : 0);
  static constexpr int kHeads = 8 * NT;
  static constexpr int kPitch = DP + 4;
  static constexpr int kScratch = static_cast<int>(sizeof(FindScratch));
  static constexpr int kFit = (228 * 1024 / 3 - 1024 - kScratch) / (kSplitWarps * kStage);
  static constexpr int kStages = kFit < 2 ? 2 : kFit > 4 ? 4 : kFit;
  static constexpr int kSmem = kSplitWarps * kStages * kStage + kScratch;
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
// e4m3: codes become fp16 in registers, q is scaled by a power of two so that the head's
// largest element lies in [2^14, 2^15), and the key's scale multiplies its score. A bf16
// element is then exact down to 2^-31 of the largest, an fp16 one down to 2^-28, and off by
// 2^-39 of the largest below that; fp32 queries enter as two fp16 parts, off by 2^-22 of the
// element or by that 2^-39. The value's scale multiplies the weight, relative to the power of
// two above the largest scale that the warp has met, rows of zeros aside (the running sums
// follow when it grows): with the 2^14 that weights are held at, a weight of 1 keeps fp16's
// full fraction while its scale is above 2^-28 of the largest.
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
  constexpr int kRows = kWarp / kChunks, kTurns = kKeys / kRows;
  extern __shared__ __align__(128) unsigned char smem[];
  auto* scratch = reinterpret_cast<FindScratch*>(smem + kSplitWarps * kS * Plan::kStage);
  const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
  const int r = lane >> 2, t = lane & 3;  // row and column pair of this lane's fragments
  const int dim = static_cast<int>(sh.lay.dim);
  const uint32_t ring = smem_u32(smem) + warp * kS * Plan::kStage;
  const int chunks_in = dim * static_cast<int>(sizeof(C)) / 16;
  const int lr = lane / kChunks, ch = lane % kChunks;  // the loader's row of a turn, and chunk

  pdl_launch_dependents();
  int64_t worker;
  int count;
  UnitPlace p = find_units(seq_lens, sh, sp, scratch, &worker, &count, err);

  // The loader runs kS - 1 units ahead, and looks up its next unit's pages one unit before
  // that: next_row / next_scale are those of this lane's key (lane % kKeys).
  UnitPlace lp = p;
  int left = count;  // units that the loader has not begun
  uint32_t next_row = kNoRow, next_scale = 0;
  unsigned bad_slots = 0;
  const auto page_size = static_cast<uint32_t>(sh.lay.page_size);
  const auto page_units = static_cast<uint32_t>(sh.lay.page_stride * sizeof(C) / 16);
  auto look_up = [&]() {
    next_row = kNoRow;
    const uint32_t pos = lp.blk * kKeys + (lane & (kKeys - 1));
    if (left <= 0 || pos >= static_cast<uint32_t>(lp.n)) return;
    const uint32_t at = sp.page_log >= 0 ? pos >> sp.page_log : pos / page_size;
    const uint32_t off = pos - at * page_size;
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
      // a turn copies kRows rows, each lane a chunk of one; whole tiles without the marks
      const uint64_t lane_byte = static_cast<uint64_t>(ch) * 16;
      if (__all_sync(kFull, next_row < kBadRow) && chunks_in == kChunks) {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
          const uint64_t byte =
              static_cast<uint64_t>(__shfl_sync(kFull, next_row, i * kRows + lr)) * 16 + lane_byte;
          const uint32_t at = tile_turn<kRow>(i * kRows, lr, ch);
          cp_async16(kd + at, reinterpret_cast<const char*>(k_cache) + byte);
          cp_async16(vd + at, reinterpret_cast<const char*>(v_cache) + byte);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
          const uint32_t row = __shfl_sync(kFull, next_row, i * kRows + lr);
          const bool in = row < kBadRow && ch < chunks_in;
          const uint64_t byte = in ? static_cast<uint64_t>(row) * 16 + lane_byte : 0;
          const uint32_t at = tile_turn<kRow>(i * kRows, lr, ch);
          cp_async16(kd + at, reinterpret_cast<const char*>(k_cache) + byte, in);
          cp_async16(vd + at, reinterpret_cast<const char*>(v_cache) + byte, in);
        }
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
      if (lp.b >= sh.batch) left = 0;
    }
    cp_async_commit();  // an empty group where nothing is left, so that the count stays
    look_up();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < kS - 1; ++i) load(i);

  constexpr int kParts = std::is_same_v<T, float> ? 2 : 1;  // 16-bit parts of q
  uint32_t qb[kParts][NT][kSteps][2];
  float mult[NT][2];                      // score -> log2 units, heads 2t and 2t + 1
  float acc[NT][kSteps][4];               // O^T: elements x heads
  float m[NT][2], l[NT][2];               // running maximum and sum
  uint32_t vref = 1;                      // e4m3: exponent that value scales are relative to
  bool fresh = true, whole_start = p.blk == 0;
  int slot = 0, stage = 0;
  for (; count > 0 && p.b < sh.batch; --count) {
    if (fresh) {
      fresh = false;
      const int64_t hk = static_cast<uint32_t>(p.row) / sp.tiles;
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
              qb[0][nt][kk][i] =
                  live && d < dim ? *reinterpret_cast<const uint32_t*>(qh + d) : 0u;
            }
          }
          mult[nt][0] = mult[nt][1] = sh.scale * kLog2e;
        } else {
          // elements 4t .. 4t+3 of each 16, in the order that a word of codes has them
          using Raw = std::conditional_t<std::is_same_v<T, float>, float4, uint2>;
          Raw raw[kSteps];
          uint32_t top = 0;
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
            const int d = kk * 16 + 4 * t;
            raw[kk] = Raw{};
            if (live && d < dim) raw[kk] = *reinterpret_cast<const Raw*>(qh + d);
            const T* e = reinterpret_cast<const T*>(&raw[kk]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              top = max(top, __float_as_uint(to_f(e[i])) & 0x7fffffffu);
          }
          top = max(top, __shfl_xor_sync(kFull, top, 1));
          top = max(top, __shfl_xor_sync(kFull, top, 2));
          // down: brings the head's largest magnitude, of exponent ex, to [2^kQueryBits,
          // 2^(kQueryBits + 1)); up = 1 / down. Both stay normal numbers: what is smaller than
          // 2^(kQueryBits - 126) is scaled by 2^126. A head that is not finite ends as NaN
          uint32_t ex = top >> 23;
          ex = ex == 255 ? 127 : max(ex, kQueryBits + 1u);
          const float down = __uint_as_float((254 + kQueryBits - ex) << 23);
          const float up = __uint_as_float((ex - kQueryBits) << 23);
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
            const T* e = reinterpret_cast<const T*>(&raw[kk]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float x = to_f(e[2 * i]) * down, y = to_f(e[2 * i + 1]) * down;
#pragma unroll
              for (int part = 0; part < kParts; ++part) {
                const __half2 v = __floats2half2_rn(x, y);
                qb[part][nt][kk][i] = *reinterpret_cast<const uint32_t*>(&v);
                x -= __low2float(v);
                y -= __high2float(v);
              }
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
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
      }
      vref = 1;
    }

    load(stage == 0 ? kS - 1 : stage - 1);
    cp_async_wait<kS - 1>();
    __syncwarp();
    const uint32_t kt = ring + stage * Plan::kStage, vt = kt + Plan::kTile;
    const int key0 = p.blk * kKeys;
    // scores: block l / 8 of an ldmatrix is keys (l / 8) % 2 * 8 .., chunk + l / 16
    const int krow = (lane & 7) + ((lane >> 3) & 1) * 8, kch = lane >> 4;
    // two chains of sums where a single 16-key tile would leave one
    constexpr int kChains = kTiles * NT > 1 ? 1 : 2;
    float c[kTiles][NT][kChains][4] = {};
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      if constexpr (!kQuant) {
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
          uint32_t a[4];
          ldmatrix4<false>(kt + tile_at<kRow>(krow + 16 * j, 2 * kk + kch), a);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<M>(c[j][nt][kk % kChains], a[0], a[1], a[2], a[3], qb[0][nt][kk][0],
                        qb[0][nt][kk][1]);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < kSteps; kk += 2) {
          uint32_t w[4];
          ldmatrix4<false>(kt + tile_at<kRow>(krow + 16 * j, kk + kch), w);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a0, a1, a2, a3;
            codes_to_half(w[2 * i], &a0, &a2);
            codes_to_half(w[2 * i + 1], &a1, &a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int part = 0; part < kParts; ++part)
                mma16816<M>(c[j][nt][i % kChains], a0, a1, a2, a3, qb[part][nt][kk + i][0],
                            qb[part][nt][kk + i][1]);
            }
          }
        }
      }
    }
    float ks[kTiles][2], vs[kTiles][2], shrink = 1.f;
    if constexpr (kQuant) {
      float* sc = reinterpret_cast<float*>(
          smem + (warp * kS + stage) * Plan::kStage + 2 * Plan::kTile);
      // the exponent above the largest finite value scale (positive: ordered as integers);
      // past the last key the scale's place holds 0
      const auto above = [](uint32_t bits) { return min((bits >> 23) + 1, 253u); };
      const int my_key = lane & (kKeys - 1);
      uint32_t mine = __float_as_uint(sc[kKeys + my_key]);
      if (mine >= 0x7f800000u) mine = 0u;
      if (above(__reduce_max_sync(kFull, mine)) > vref) {
        // a row of zeros has the scale 1, however small the others are: it counts as 0
        const unsigned char* values = smem + (warp * kS + stage) * Plan::kStage + Plan::kTile;
        if (above(mine) > vref && row_is_zero<kRow>(values, my_key)) sc[kKeys + my_key] = mine = 0;
        __syncwarp();
        const uint32_t top = above(__reduce_max_sync(kFull, mine));
        if (top > vref) {  // the sums so far become relative to the new one
          shrink = exp2f(static_cast<float>(static_cast<int>(vref) - static_cast<int>(top)));
          vref = top;
        }
      }
      const float down = __uint_as_float((254 - vref) << 23);
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ks[j][h] = sc[16 * j + 8 * h + r];
          vs[j][h] = sc[kKeys + 16 * j + 8 * h + r] * down;
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
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float s = c[j][nt][0][2 * h + i];
            if constexpr (kChains == 2) s += c[j][nt][1][2 * h + i];
            s *= kQuant ? mult[nt][i] * ks[j][h] : mult[nt][i];
            if (!full && key0 + 16 * j + 8 * h + r >= p.n) s = -INFINITY;
            w[j][h][i] = s;
            top = fmaxf(top, s);
          }
        }
#pragma unroll
        for (int off = 4; off < kWarp; off <<= 1)
          top = fmaxf(top, __shfl_xor_sync(kFull, top, off));
        const float m_new = fmaxf(m[nt][i], top);
        const float base = m_new == -INFINITY ? 0.f : m_new;
        alpha[i] = ex2f(m[nt][i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            w[j][h][i] = ex2f(w[j][h][i] - (base - kWeightBits<M>));
            sum += w[j][h][i];
            if constexpr (kQuant) w[j][h][i] *= vs[j][h];
          }
        }
        l[nt][i] = fmaf(l[nt][i], alpha[i], sum);
        m[nt][i] = m_new;
        if constexpr (kQuant) alpha[i] *= shrink;
      }
      if (__any_sync(kFull, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][kk][i] *= alpha[i & 1];
        }
      }
      // fp16: a weight below kHalfTiny (26 nats below the largest and more) is cut to 0, which
      // is wrong beside an infinite value only: the tile is searched where there are any, and
      // such weights raised to kHalfTiny beside one
      if constexpr (!kQuant && std::is_same_v<M, __half>) {
        uint32_t least = 0xffffffffu;  // bits - 1 of the smallest weight above 0
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 2; ++i) least = min(least, __float_as_uint(w[j][h][i]) - 1u);
          }
        }
        if (__any_sync(kFull, least < __float_as_uint(kHalfTiny) - 1u) &&
            tile_has_inf(smem + (warp * kS + stage) * Plan::kStage + Plan::kTile, Plan::kTile)) {
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int i = 0; i < 2; ++i)
                w[j][h][i] = w[j][h][i] > 0.f ? fmaxf(w[j][h][i], kHalfTiny) : w[j][h][i];
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t rest;
          hi[j][nt][h] = transpose8(split_weights<M, !kQuant>(w[j][h][0], w[j][h][1], &rest));
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
            uint32_t a0, a1, a2, a3;
            codes_to_half(__byte_perm(w[2 * i], 0, 0x3120), &a0, &a1);
            codes_to_half(__byte_perm(w[2 * i + 1], 0, 0x3120), &a2, &a3);
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
    __syncwarp();  // every lane has read this stage before it is filled again
    stage = stage + 1 == kS ? 0 : stage + 1;

    const bool row_ends = p.blk + 1 == p.blocks;
    if (row_ends || count == 1) {
      const bool whole = whole_start && row_ends;
      if (whole_start && lane == 0) note_shared(p, whole, worker, slot, count, scratch, sp);
      const int64_t hk = static_cast<uint32_t>(p.row) / sp.tiles;
      const int first = static_cast<int>(p.row - hk * sp.tiles) * kHeads;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float sum = l[nt][i];
#pragma unroll
          for (int off = 4; off < kWarp; off <<= 1) sum += __shfl_xor_sync(kFull, sum, off);
          const int h = nt * 8 + 2 * t + i;
          if (first + h < sp.group) {
            // out of the weights' units, and of 2^(vref - 127) for e4m3 values: one after the
            // other, since the product of the two may leave fp32's range
            const float f = whole ? 1.f / sum : kWeightUnit<M>;
            const float vf = kQuant ? __uint_as_float(vref << 23) : 1.f;
            T* out = o + (p.b * sh.q_heads + hk * sp.group + first + h) * dim;
            float* part = partial_at(sp, worker, slot, h);
            if (!whole && r == 0) {
              part[DP] = m[nt][i];
              part[DP + 1] = sum * f;
            }
#pragma unroll
            for (int kk = 0; kk < kSteps; ++kk) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int d = kk * 16 + (kQuant ? 2 * r + j : r + 8 * j);
                const float v = acc[nt][kk][2 * j + i] * f * vf;
                if (!whole) part[d] = v;
                else if (d < dim) out[d] = from_f<T>(v);
              }
            }
          }
        }
      }
      fresh = true;
      whole_start = true;
      slot = 1;
    }
    p.next(seq_lens, sh, sp, err);
  }
  cp_async_wait<0>();
  zero_empty(o, seq_lens, sh, sp, err);
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

int64_t partial_floats(int tile_heads, int pitch) {
  return int64_t{2} * tile_heads * pitch;
}

size_t notes_bytes(int64_t rows) {
  return static_cast<size_t>(cdiv(rows * static_cast<int64_t>(sizeof(int2)), 16) * 16);
}

// Units of a call if every sequence were as long as its table allows.
int64_t units_bound(int64_t batch, int64_t rows, int64_t max_len, int unit) {
  const int64_t per = cdiv(max_len, unit) * rows;
  return per == 0 ? 0 : batch > INT64_MAX / 4096 / per ? INT64_MAX / 4096 : batch * per;
}

// Grid of the first kernel: one wave of `per_sm` CTAs an SM, no more than units.
int64_t split_ctas(int64_t units, int per_sm) {
  return std::max<int64_t>(1, std::min<int64_t>(units, int64_t{per_sm} * sm_count()));
}

// CTAs an SM at most: what the sums' registers leave, and what bounds the partials.
constexpr int kMmaCtasPerSm = 4;
constexpr int simt_ctas_per_sm(int heads) { return heads >= 4 ? 4 : 8; }

template <typename T, int E>
int launch_join(const PagedCall& c, const SplitShape& sp, int64_t workers) {
  const int64_t max_len = c.sh.max_pages * c.sh.lay.page_size;
  if (max_len <= int64_t{1} << sp.deal_log) return KPB_OK;  // no row is dealt out in parts
  cudaLaunchConfig_t cfg = {};
  // warps per head: enough for 16 an SM where heads are few, one where they are many
  const int64_t heads = c.sh.batch * c.sh.q_heads;  // below 2^31
  int share_log = 0;
  while (2 << share_log <= kJoinWarps && (heads << (share_log + 1)) <= int64_t{16} * sm_count())
    ++share_log;
  cfg.gridDim = dim3(static_cast<unsigned>(cdiv(heads, kJoinWarps >> share_log)));
  cfg.blockDim = dim3(kJoinWarps * kWarp);
  cfg.stream = c.s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  KPB_CUDA(cudaLaunchKernelEx(&cfg, join_rows<T, E>, static_cast<T*>(c.o),
                              static_cast<int>(heads), static_cast<int>(c.sh.lay.dim), sp,
                              static_cast<int>(workers), share_log));
  return KPB_OK;
}

// Rows of a table of up to `whole` keys are not dealt out in parts.
SplitShape split_shape(const PagedCall& c, int tile_heads, int pitch, int unit, int whole,
                       void* ws) {
  SplitShape sp;
  sp.group = static_cast<int>(c.sh.q_heads / c.sh.lay.heads);
  sp.tile_heads = tile_heads;
  sp.tiles = static_cast<int>(cdiv(sp.group, tile_heads));
  sp.rows = c.sh.lay.heads * sp.tiles;
  sp.pitch = pitch;
  sp.unit_log = log2_of(unit);
  const int64_t max_len = c.sh.max_pages * c.sh.lay.page_size;
  sp.deal_log = max_len <= whole ? log2_of(whole) : sp.unit_log;
  sp.page_log = log2_of(c.sh.lay.page_size);
  sp.shared = static_cast<int2*>(ws);
  sp.partials =
      reinterpret_cast<float*>(static_cast<char*>(ws) + notes_bytes(c.sh.batch * sp.rows));
  return sp;
}

template <typename T, typename C, int E, int HG, bool kRing>
int launch_simt(const PagedCall& c, void* ws) {
  const SplitShape sp = split_shape(c, HG, E * kWarp + 4, kSimtUnit, kSimtUnit, ws);
  auto* kernel = split_simt<T, C, E, HG, kRing>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  constexpr int kSmem = kRing ? simt_ring_bytes(E) : 0;
  if (kSmem > 0) {
    if (int rc = ensure_dyn_smem(fn, kSmem)) return rc;
  }
  int occ = 0;
  if (int rc = occupancy_blocks(fn, kSplitThreads, kSmem, &occ)) return rc;
  const int64_t units =
      units_bound(c.sh.batch, sp.rows, c.sh.max_pages * c.sh.lay.page_size, kSimtUnit);
  const int64_t ctas = split_ctas(units, std::min(occ, simt_ctas_per_sm(HG)));
  kernel<<<static_cast<unsigned>(ctas), kSplitThreads, kSmem, c.s>>>(
      static_cast<const T*>(c.q), static_cast<const C*>(c.k_cache),
      static_cast<const C*>(c.v_cache), c.table, c.seq_lens, c.k_scale, c.v_scale,
      static_cast<T*>(c.o), c.sh, sp, c.err);
  KPB_LAUNCHED("paged_attention split");
  return launch_join<T, E>(c, sp, std::min(units, ctas * kSplitWarps));
}

template <typename T, typename C, int E, int HG>
int dispatch_simt_ring(const PagedCall& c, void* ws) {
  if constexpr (std::is_same_v<C, float>) {
    constexpr int VE = simt_vector(E);
    const uintptr_t both =
        reinterpret_cast<uintptr_t>(c.k_cache) | reinterpret_cast<uintptr_t>(c.v_cache);
    if (c.sh.lay.dim % VE == 0 && both % (VE * 4) == 0 &&
        (c.sh.lay.num_pages < 2 || c.sh.lay.page_stride % VE == 0))
      return launch_simt<T, C, E, HG, true>(c, ws);
  }
  return launch_simt<T, C, E, HG, false>(c, ws);
}

// Heads per tile: the smallest of 1, 2, 4, 8 that holds the group, 8 for larger ones.
template <typename T, typename C, int E>
int dispatch_simt_heads(const PagedCall& c, void* ws) {
  const int64_t group = c.sh.q_heads / c.sh.lay.heads;
  if (group <= 1) return dispatch_simt_ring<T, C, E, 1>(c, ws);
  if (group <= 2) return dispatch_simt_ring<T, C, E, 2>(c, ws);
  if (group <= 4) return dispatch_simt_ring<T, C, E, 4>(c, ws);
  return dispatch_simt_ring<T, C, E, 8>(c, ws);
}

template <typename T, typename C>
int dispatch_simt(const PagedCall& c, void* ws) {
  if (c.sh.lay.dim <= 64) return dispatch_simt_heads<T, C, 2>(c, ws);
  if (c.sh.lay.dim <= 128) return dispatch_simt_heads<T, C, 4>(c, ws);
  return dispatch_simt_heads<T, C, 8>(c, ws);
}

// Where no sequence can have more than 64 keys a warp takes whole rows: their two to four
// units take it less time than a second kernel takes to join them (one sequence of 32 keys
// 6.4 us and not 8.0, of 64 the same; 64 sequences 7.0 and not 9.5, 8.8 and not 11.2). On
// the CUDA cores a unit takes longer (one sequence of 64 fp32 keys 15.3 us and not 9.7).
constexpr int kWholeRow = 64;

template <typename T, typename C, int DP, int NT>
int launch_mma(const PagedCall& c, void* ws) {
  using Plan = MmaPlan<C, DP, NT>;
  const SplitShape sp = split_shape(c, Plan::kHeads, Plan::kPitch, Plan::kKeys, kWholeRow, ws);
  auto* kernel = split_mma<T, C, DP, NT>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  if (int rc = ensure_dyn_smem(fn, Plan::kSmem)) return rc;
  int occ = 0;
  if (int rc = occupancy_blocks(fn, kSplitThreads, Plan::kSmem, &occ)) return rc;
  const int64_t units =
      units_bound(c.sh.batch, sp.rows, c.sh.max_pages * c.sh.lay.page_size, Plan::kKeys);
  const int64_t ctas = split_ctas(units, std::min(occ, kMmaCtasPerSm));
  kernel<<<static_cast<unsigned>(ctas), kSplitThreads, Plan::kSmem, c.s>>>(
      static_cast<const T*>(c.q), static_cast<const C*>(c.k_cache),
      static_cast<const C*>(c.v_cache), c.table, c.seq_lens, c.k_scale, c.v_scale,
      static_cast<T*>(c.o), c.sh, sp, c.err);
  KPB_LAUNCHED("paged_attention split");
  return launch_join<T, DP / kWarp>(c, sp, std::min(units, ctas * kSplitWarps));
}

template <typename T, typename C>
int dispatch_mma_16(const PagedCall& c, void* ws) {
  const bool wide = c.sh.q_heads / c.sh.lay.heads > 8;
  if (c.sh.lay.dim <= 64)
    return wide ? launch_mma<T, C, 64, 2>(c, ws) : launch_mma<T, C, 64, 1>(c, ws);
  if (c.sh.lay.dim <= 128)
    return wide ? launch_mma<T, C, 128, 2>(c, ws) : launch_mma<T, C, 128, 1>(c, ws);
  return launch_mma<T, C, 256, 1>(c, ws);
}

// Sixteen heads to a tile where the group has more than eight, so that its keys are read
// once; at D > 128, and with the two parts of fp32 queries, they would not fit the registers.
template <typename T, typename C>
int dispatch_mma(const PagedCall& c, void* ws) {
  if constexpr (std::is_same_v<T, float>) {
    return c.sh.lay.dim <= 64 ? launch_mma<T, C, 64, 1>(c, ws) : launch_mma<T, C, 128, 1>(c, ws);
  } else {
    return dispatch_mma_16<T, C>(c, ws);
  }
}

// Rows of the cache whole 16-byte chunks on 16-byte boundaries (cp.async), four elements of q
// on theirs; the cache's 16-byte units counted in 32 bits (64 GB, of 180 on the card).
template <typename T, typename C>
bool mma_takes(const PagedCall& c) {
  const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const KvLayout& lay = c.sh.lay;
  const int64_t extent = (lay.num_pages < 2 ? 0 : (lay.num_pages - 1) * lay.page_stride) +
                         lay.heads * lay.page_size * lay.dim;
  return lay.dim * sizeof(C) % 16 == 0 && lay.dim % 8 == 0 &&
         (at(c.k_cache) | at(c.v_cache)) % 16 == 0 &&
         (lay.num_pages < 2 || lay.page_stride * sizeof(C) % 16 == 0) &&
         static_cast<int64_t>(extent * sizeof(C) / 16) < kBadRow &&
         at(c.q) % (4 * sizeof(T)) == 0 && (c.sh.batch < 2 || c.sh.q_stride % 4 == 0);
}

template <typename T, typename C>
int launch(int variant, const PagedCall& c, void* ws) {
  if (variant == 0 || c.sh.lay.num_pages == 0) {  // no page to point a copy at
    paged_cta_head<T, C><<<static_cast<unsigned>(c.sh.batch * c.sh.q_heads), 128, 0, c.s>>>(
        static_cast<const T*>(c.q), static_cast<const C*>(c.k_cache),
        static_cast<const C*>(c.v_cache), c.table, c.seq_lens, c.k_scale, c.v_scale,
        static_cast<T*>(c.o), c.sh, c.err);
    KPB_LAUNCHED("paged_attention variant 0");
    return KPB_OK;
  }
  // fp32 keys and values have no product that keeps their bits; e4m3 codes are exact in fp16
  if constexpr (sizeof(T) == 2 || sizeof(C) == 1) {
    if (mma_takes<T, C>(c) && (sizeof(T) == 2 || c.sh.lay.dim <= 128))
      return dispatch_mma<T, C>(c, ws);
  }
  return dispatch_simt<T, C>(c, ws);
}

}  // namespace

size_t paged_attention_workspace_bytes(int variant, int64_t batch, int64_t q_heads,
                                       int64_t k_heads, int64_t dim, int64_t max_len) {
  if (variant == 0) return 0;
  // the widest tile and pitch that either way takes for this call, and as many workers as
  // there can be warps and units (a tile holds one head at least, a unit 16 keys); the
  // CUDA-core way has twice the CTAs for tiles of a quarter of the heads
  const int pitch = static_cast<int>(dim <= 64 ? 64 : dim <= 128 ? 128 : 256) + 4;
  const int heads = q_heads / k_heads > 8 && dim <= 128 ? 16 : 8;
  const int64_t units = units_bound(batch, q_heads, max_len, kSimtUnit);
  const int64_t workers = std::min(units, kSplitWarps * split_ctas(units, kMmaCtasPerSm));
  return notes_bytes(batch * q_heads) +
         static_cast<size_t>(workers * partial_floats(heads, pitch)) * sizeof(float);
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
      return e4m3 ? launch<__half, uint8_t>(variant, c, ws)
                  : launch<__half, __half>(variant, c, ws);
    default:
      return e4m3 ? launch<__nv_bfloat16, uint8_t>(variant, c, ws)
                  : launch<__nv_bfloat16, __nv_bfloat16>(variant, c, ws);
  }
}

}  // namespace kpb
