// The extern "C" boundary (include/kp_b200.h): argument validation, status codes,
// per-thread error messages, stream-ordered scratch from a pool of its own, and the
// per-device error word that bounded waits inside kernels report timeouts to.
#include <map>
#include <mutex>
#include <string>
#include <tuple>

#include "kp_common.cuh"
#include "kp_kv_cache.cuh"

namespace kpb {

// implemented by the kernel translation units
size_t reduce_workspace_bytes(int variant, int64_t n);
int reduce_sum(int variant, int dtype, const void* x, float* out, int64_t n, void* ws,
               size_t ws_bytes, cudaStream_t s);
int softmax(int variant, int dtype, const void* x, void* y, int64_t M, int64_t N,
            unsigned* err, cudaStream_t s);
size_t matmul_workspace_bytes(int variant, int dtype, int64_t M, int64_t N, int64_t K);
int matmul(int variant, int dtype, const void* A, const void* B, void* C, int64_t M, int64_t N,
           int64_t K, void* ws, size_t ws_bytes, unsigned* err, cudaStream_t s);
int vector_add(int variant, int dtype, const void* a, const void* b, void* c, int64_t n,
               cudaStream_t s);
int layernorm(int variant, int dtype, const void* x, const void* w, const void* b, void* y,
              int64_t M, int64_t N, float eps, cudaStream_t s);
int attention(int variant, int dtype, bool causal, const void* q, const void* k, const void* v,
              void* o, int64_t BH, int64_t S, int64_t D, unsigned* err, cudaStream_t s);
int qk_norm_rope(int variant, int dtype, const void* q, const void* k, const void* wq,
                 const void* wk, const float* cos_sin, const int64_t* positions, void* q_out,
                 void* k_out, int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t dim,
                 int64_t rot, int64_t max_pos, int64_t q_stride, int64_t k_stride, float eps,
                 bool interleaved, unsigned* err, cudaStream_t s);
size_t qk_norm_rope_backward_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t k_heads,
                                             int64_t dim);
int qk_norm_rope_backward(int variant, int dtype, const void* gq, const void* gk, const void* q,
                          const void* k, const void* wq, const void* wk, const float* cos_sin,
                          const int64_t* positions, void* dq, void* dk, void* dwq, void* dwk,
                          int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t dim,
                          int64_t rot, int64_t max_pos, int64_t gq_stride, int64_t gk_stride,
                          int64_t q_stride, int64_t k_stride, float eps, bool interleaved,
                          void* ws, unsigned* err, cudaStream_t s);
int kv_cache_write(int variant, int dtype, int cache_dtype, const void* k, const void* v,
                   const int64_t* slots, void* k_cache, void* v_cache, float* k_scale,
                   float* v_scale, int64_t tokens, int64_t k_stride, int64_t v_stride,
                   const KvLayout& lay, unsigned* err, cudaStream_t s);
int kv_cache_read(int variant, int dtype, int cache_dtype, const void* k_cache,
                  const void* v_cache, const int64_t* slots, const float* k_scale,
                  const float* v_scale, void* k, void* v, int64_t tokens, const KvLayout& lay,
                  unsigned* err, cudaStream_t s);
size_t paged_attention_workspace_bytes(int variant, int64_t batch, int64_t q_heads,
                                       int64_t k_heads, int64_t dim, int64_t max_len);
int paged_attention(int variant, int dtype, int cache_dtype, const void* q, const void* k_cache,
                    const void* v_cache, const int* table, const int* seq_lens,
                    const float* k_scale, const float* v_scale, void* o, int64_t batch,
                    int64_t q_heads, int64_t max_pages, int64_t q_stride, int64_t table_stride,
                    float scale, const KvLayout& lay, void* ws, size_t ws_bytes, unsigned* err,
                    cudaStream_t s);

namespace {
thread_local std::string g_last_error;

constexpr int kMaxDevices = 64;
std::mutex g_mu;
int g_sms[kMaxDevices] = {0};
unsigned* g_err_ptr[kMaxDevices] = {nullptr};

// Set by kernels whose bounded waits gave up (kErrTimeout); read by kpb_device_errors.
__device__ unsigned g_device_error_word = 0;
}  // namespace

void set_error(const std::string& msg) { g_last_error = msg; }

int fail(int code, const std::string& msg) {
  g_last_error = msg;
  return code;
}

int cuda_fail(cudaError_t err, const char* what, const char* file, int line) {
  g_last_error = std::string("CUDA error ") + cudaGetErrorName(err) + " (" +
                 cudaGetErrorString(err) + ") in " + what + " at " + file + ":" +
                 std::to_string(line);
  return KPB_ECUDA;
}

int sm_count() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 148;
  std::lock_guard<std::mutex> lk(g_mu);
  if (g_sms[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
    g_sms[dev] = n;
  }
  return g_sms[dev];
}

// Scratch of the allocating entry points comes from a stream-ordered pool per device
// owned by this library, which keeps its memory between calls (release threshold
// unlimited). The device's default pool returns its memory at every synchronisation,
// so the next call would map it again on the host after the GPU had already reached
// the call, and the GPU would wait for it.
namespace {
cudaMemPool_t g_pool[kMaxDevices] = {};
}  // namespace

int scratch_alloc(void** p, size_t bytes, cudaStream_t s) {
  int dev = 0;
  KPB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail(KPB_EUNSUPPORTED, "device index out of range");
  cudaMemPool_t pool = nullptr;
  {
    std::lock_guard<std::mutex> lk(g_mu);
    if (g_pool[dev] == nullptr) {
      cudaMemPoolProps props = {};
      props.allocType = cudaMemAllocationTypePinned;
      props.location.type = cudaMemLocationTypeDevice;
      props.location.id = dev;
      cudaMemPool_t created = nullptr;
      KPB_CUDA(cudaMemPoolCreate(&created, &props));
      uint64_t keep = UINT64_MAX;
      const cudaError_t e = cudaMemPoolSetAttribute(created, cudaMemPoolAttrReleaseThreshold, &keep);
      if (e != cudaSuccess) {
        cudaMemPoolDestroy(created);
        return cuda_fail(e, "cudaMemPoolSetAttribute", __FILE__, __LINE__);
      }
      g_pool[dev] = created;
    }
    pool = g_pool[dev];
  }
  KPB_CUDA(cudaMallocFromPoolAsync(p, bytes, pool, s));
  return KPB_OK;
}

// Launch facts of a kernel that do not change within a process, per device: the
// dynamic shared-memory opt-in is only raised when a launch needs more, and each
// occupancy answer is queried once for its block size, shared memory and cluster size
// (a whole launch call then costs 6-15 us of host time, with or without the cache).
namespace {
enum class Fact { kSmemOptIn, kBlocksPerSm, kClusters };
// (device, kernel, fact, threads, dynamic shared memory, cluster size)
using LaunchKey = std::tuple<int, const void*, Fact, int, size_t, int>;
std::map<LaunchKey, int> g_launch_facts;

int current_device(int* dev) {
  KPB_CUDA(cudaGetDevice(dev));
  return KPB_OK;
}
}  // namespace

// The opt-in is one value per kernel and device, and a launch may use any amount up
// to it: it is only ever raised, to the largest amount asked for so far.
int ensure_dyn_smem(const void* func, int bytes) {
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  const LaunchKey key{dev, func, Fact::kSmemOptIn, 0, 0, 0};
  std::lock_guard<std::mutex> lk(g_mu);
  auto it = g_launch_facts.find(key);
  if (it != g_launch_facts.end() && it->second >= bytes) return KPB_OK;
  KPB_CUDA(cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  g_launch_facts[key] = bytes;
  return KPB_OK;
}

int occupancy_blocks(const void* func, int threads, size_t smem, int* out) {
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  const LaunchKey key{dev, func, Fact::kBlocksPerSm, threads, smem, 0};
  std::lock_guard<std::mutex> lk(g_mu);
  auto it = g_launch_facts.find(key);
  if (it == g_launch_facts.end()) {
    int occ = 0;
    KPB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, func, threads, smem));
    it = g_launch_facts.emplace(key, occ).first;
  }
  *out = it->second;
  return KPB_OK;
}

int occupancy_clusters(const void* func, const cudaLaunchConfig_t& cfg, int cluster, int* out) {
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  const LaunchKey key{dev, func, Fact::kClusters, static_cast<int>(cfg.blockDim.x),
                      cfg.dynamicSmemBytes, cluster};
  std::lock_guard<std::mutex> lk(g_mu);
  auto it = g_launch_facts.find(key);
  if (it == g_launch_facts.end()) {
    int active = 0;
    KPB_CUDA(cudaOccupancyMaxActiveClusters(&active, func, &cfg));
    it = g_launch_facts.emplace(key, active).first;
  }
  *out = it->second;
  return KPB_OK;
}

// Device address of this device's error word (looked up once per device).
int device_error_word(unsigned** out) {
  int dev = 0;
  KPB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail(KPB_EUNSUPPORTED, "device index out of range");
  std::lock_guard<std::mutex> lk(g_mu);
  if (g_err_ptr[dev] == nullptr) {
    void* p = nullptr;
    KPB_CUDA(cudaGetSymbolAddress(&p, g_device_error_word));
    g_err_ptr[dev] = static_cast<unsigned*>(p);
  }
  *out = g_err_ptr[dev];
  return KPB_OK;
}

static bool valid_dtype(int dt) { return dt == KPB_F32 || dt == KPB_F16 || dt == KPB_BF16; }

static int check_common(const char* op, int variant, int dtype) {
  const int nv = kpb_num_variants(op);
  if (variant < 0 || variant >= nv)
    return fail(KPB_EINVAL, std::string(op) + ": variant must be in [0, " + std::to_string(nv) +
                                ")");
  if (!valid_dtype(dtype))
    return fail(KPB_EINVAL, std::string(op) + ": dtype must be 0 (f32), 1 (f16) or 2 (bf16)");
  return KPB_OK;
}

static size_t elem_bytes(int dtype) { return dtype == KPB_F32 ? 4 : 2; }

constexpr int64_t kSizeLimit = int64_t{1} << 31;

static bool size_ok(int64_t n) { return n >= 0 && n < kSizeLimit; }

static bool off_by(const void* p, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes != 0;
}

// Sizes of qk_norm_rope and its backward.
static int check_rope(const std::string& op, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                      int64_t rot, int64_t max_pos) {
  if (!size_ok(T) || !size_ok(Hq) || !size_ok(Hkv) || !size_ok(max_pos) ||
      !size_ok(T * (Hq + Hkv)))
    return fail(KPB_EINVAL, op + ": T, heads, T * heads and max_pos must be in [0, 2^31)");
  if (D < 1 || D > kMaxHeadDim) return fail(KPB_EINVAL, op + ": D must be in [1, 256]");
  if (rot < 0 || rot > D || rot % 2 != 0)
    return fail(KPB_EINVAL, op + ": rot must be even and in [0, D]");
  return KPB_OK;
}

// Sizes, types and strides of a paged cache.
static int check_cache(const std::string& op, int dtype, int cache_dtype, const void* k_cache,
                       const void* v_cache, const void* k_scale, const void* v_scale,
                       const KvLayout& lay) {
  if (cache_dtype != dtype && cache_dtype != KPB_E4M3)
    return fail(KPB_EINVAL, op + ": cache dtype must be the call's dtype or 3 (e4m3)");
  if (!size_ok(lay.num_pages) || !size_ok(lay.page_size) || lay.page_size < 1 ||
      !size_ok(lay.heads))
    return fail(KPB_EINVAL,
                op + ": num_pages and Hkv must be in [0, 2^31), page_size in [1, 2^31)");
  if (lay.dim < 1 || lay.dim > kMaxHeadDim)
    return fail(KPB_EINVAL, op + ": D must be in [1, 256]");
  if (!size_ok(lay.heads * lay.page_size))
    return fail(KPB_EINVAL, op + ": Hkv * page_size must be below 2^31");
  if (lay.num_pages > 1 && lay.page_stride < lay.heads * lay.page_size * lay.dim)
    return fail(KPB_EINVAL, op + ": page_stride is shorter than a page");
  if (lay.num_pages > 0 && lay.page_stride > INT64_MAX / 16 / lay.num_pages)
    return fail(KPB_EINVAL, op + ": the cache is too large");
  const bool any = lay.num_pages > 0 && lay.heads > 0;
  if (any && (k_cache == nullptr || v_cache == nullptr))
    return fail(KPB_EINVAL, op + ": null pointer");
  if (cache_dtype == KPB_E4M3) {
    if (any && (k_scale == nullptr || v_scale == nullptr))
      return fail(KPB_EINVAL, op + ": an e4m3 cache needs k_scale and v_scale (null pointer)");
    if (off_by(k_scale, 4) || off_by(v_scale, 4))
      return fail(KPB_EINVAL, op + ": scales must be element-aligned");
  } else if (off_by(k_cache, elem_bytes(dtype)) || off_by(v_cache, elem_bytes(dtype))) {
    return fail(KPB_EINVAL, op + ": tensors must be element-aligned");
  }
  return KPB_OK;
}

}  // namespace kpb

using namespace kpb;

extern "C" {

const char* kpb_last_error(void) { return g_last_error.c_str(); }

int kpb_version(void) { return 101; }

int kpb_num_variants(const char* op) {
  if (op == nullptr) return -1;
  const std::string s(op);
  if (s == "vector_add" || s == "reduce_sum" || s == "softmax" || s == "layernorm") return 3;
  if (s == "matmul") return 4;
  if (s == "attention" || s == "attention_causal") return 2;
  if (s == "qk_norm_rope" || s == "qk_norm_rope_backward" || s == "kv_cache_write" ||
      s == "kv_cache_read" || s == "paged_attention")
    return 2;
  return -1;
}

int kpb_device_errors(unsigned* bits) {
  g_last_error.clear();
  unsigned v = 0, zero = 0;
  KPB_CUDA(cudaMemcpyFromSymbol(&v, g_device_error_word, sizeof(v)));
  KPB_CUDA(cudaMemcpyToSymbol(g_device_error_word, &zero, sizeof(zero)));
  if (bits) *bits = v;
  return KPB_OK;
}

int kpb_vector_add(int variant, int dtype, const void* a, const void* b, void* c, int64_t n,
                   void* stream) {
  g_last_error.clear();
  if (int rc = check_common("vector_add", variant, dtype)) return rc;
  if (n < 0) return fail(KPB_EINVAL, "vector_add: n must be >= 0");
  if (n > 0 && (a == nullptr || b == nullptr || c == nullptr))
    return fail(KPB_EINVAL, "vector_add: null pointer");
  return vector_add(variant, dtype, a, b, c, n, static_cast<cudaStream_t>(stream));
}

size_t kpb_reduce_sum_workspace_bytes(int variant, int64_t n) {
  return reduce_workspace_bytes(variant, n);
}

int kpb_reduce_sum_ws(int variant, int dtype, const void* x, float* out, int64_t n,
                      void* workspace, size_t workspace_bytes, void* stream) {
  g_last_error.clear();
  if (int rc = check_common("reduce_sum", variant, dtype)) return rc;
  if (n < 0) return fail(KPB_EINVAL, "reduce_sum: n must be >= 0");
  if (out == nullptr || (n > 0 && x == nullptr))
    return fail(KPB_EINVAL, "reduce_sum: null pointer");
  return reduce_sum(variant, dtype, x, out, n, workspace, workspace_bytes,
                    static_cast<cudaStream_t>(stream));
}

int kpb_reduce_sum(int variant, int dtype, const void* x, float* out, int64_t n, void* stream) {
  g_last_error.clear();
  if (int rc = check_common("reduce_sum", variant, dtype)) return rc;
  if (n < 0) return fail(KPB_EINVAL, "reduce_sum: n must be >= 0");
  if (out == nullptr || (n > 0 && x == nullptr))
    return fail(KPB_EINVAL, "reduce_sum: null pointer");
  auto s = static_cast<cudaStream_t>(stream);
  const size_t bytes = reduce_workspace_bytes(variant, n);
  void* ws = nullptr;
  if (bytes) {
    if (int rc = scratch_alloc(&ws, bytes, s)) return rc;
  }
  const int rc = reduce_sum(variant, dtype, x, out, n, ws, bytes, s);
  if (ws) {
    const cudaError_t e = cudaFreeAsync(ws, s);
    if (rc == KPB_OK && e != cudaSuccess) return cuda_fail(e, "cudaFreeAsync", __FILE__, __LINE__);
  }
  return rc;
}

int kpb_softmax(int variant, int dtype, const void* x, void* y, int64_t M, int64_t N,
                void* stream) {
  g_last_error.clear();
  if (int rc = check_common("softmax", variant, dtype)) return rc;
  if (M < 0 || N < 0 || M >= (int64_t{1} << 31) || N >= (int64_t{1} << 31))
    return fail(KPB_EINVAL, "softmax: M and N must be in [0, 2^31)");
  if (M * N > 0 && (x == nullptr || y == nullptr)) return fail(KPB_EINVAL, "softmax: null pointer");
  unsigned* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return softmax(variant, dtype, x, y, M, N, err, static_cast<cudaStream_t>(stream));
}

int kpb_layernorm(int variant, int dtype, const void* x, const void* w, const void* b, void* y,
                  int64_t M, int64_t N, float eps, void* stream) {
  g_last_error.clear();
  if (int rc = check_common("layernorm", variant, dtype)) return rc;
  if (M < 0 || N < 0 || M >= (int64_t{1} << 31) || N >= (int64_t{1} << 31))
    return fail(KPB_EINVAL, "layernorm: M and N must be in [0, 2^31)");
  if (M * N > 0 && (x == nullptr || w == nullptr || b == nullptr || y == nullptr))
    return fail(KPB_EINVAL, "layernorm: null pointer");
  return layernorm(variant, dtype, x, w, b, y, M, N, eps, static_cast<cudaStream_t>(stream));
}

size_t kpb_matmul_workspace_bytes(int variant, int dtype, int64_t M, int64_t N, int64_t K) {
  if (!valid_dtype(dtype) || M < 0 || N < 0 || K < 0) return 0;
  return matmul_workspace_bytes(variant, dtype, M, N, K);
}

int kpb_matmul_ws(int variant, int dtype, const void* A, const void* B, void* C, int64_t M,
                  int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  g_last_error.clear();
  if (int rc = check_common("matmul", variant, dtype)) return rc;
  const int64_t lim = int64_t{1} << 31;
  if (M < 0 || N < 0 || K < 0 || M >= lim || N >= lim || K >= lim)
    return fail(KPB_EINVAL, "matmul: M, N, K must be in [0, 2^31)");
  if (M * N > 0 && (C == nullptr || (K > 0 && (A == nullptr || B == nullptr))))
    return fail(KPB_EINVAL, "matmul: null pointer");
  auto s = static_cast<cudaStream_t>(stream);
  if (M == 0 || N == 0) return KPB_OK;
  if (K == 0) {
    KPB_CUDA(cudaMemsetAsync(C, 0, static_cast<size_t>(M * N) * elem_bytes(dtype), s));
    return KPB_OK;
  }
  unsigned* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return matmul(variant, dtype, A, B, C, M, N, K, workspace, workspace_bytes, err, s);
}

int kpb_matmul(int variant, int dtype, const void* A, const void* B, void* C, int64_t M,
               int64_t N, int64_t K, void* stream) {
  g_last_error.clear();
  if (int rc = check_common("matmul", variant, dtype)) return rc;
  if (M < 0 || N < 0 || K < 0) return fail(KPB_EINVAL, "matmul: negative size");
  auto s = static_cast<cudaStream_t>(stream);
  const size_t bytes = matmul_workspace_bytes(variant, dtype, M, N, K);
  void* ws = nullptr;
  if (bytes) {
    if (int rc = scratch_alloc(&ws, bytes, s)) return rc;
  }
  const int rc = kpb_matmul_ws(variant, dtype, A, B, C, M, N, K, ws, bytes, stream);
  if (ws) {
    const std::string msg = g_last_error;
    const cudaError_t e = cudaFreeAsync(ws, s);
    if (rc == KPB_OK && e != cudaSuccess) return cuda_fail(e, "cudaFreeAsync", __FILE__, __LINE__);
    g_last_error = msg;
  }
  return rc;
}

static int attention_entry(const char* op, bool causal, int variant, int dtype, const void* q,
                           const void* k, const void* v, void* o, int64_t BH, int64_t S,
                           int64_t D, void* stream) {
  g_last_error.clear();
  if (int rc = check_common(op, variant, dtype)) return rc;
  if (BH < 0 || S < 0 || D < 0) return fail(KPB_EINVAL, std::string(op) + ": negative size");
  if (D > 256 || BH >= 65536)
    return fail(KPB_EINVAL, std::string(op) + ": supports D <= 256 and B*H < 65536");
  if (S >= (int64_t{1} << 31)) return fail(KPB_EINVAL, std::string(op) + ": S too large");
  if (BH * S * D > 0 && (!q || !k || !v || !o))
    return fail(KPB_EINVAL, std::string(op) + ": null pointer");
  if (BH == 0 || S == 0 || D == 0) return KPB_OK;
  unsigned* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return attention(variant, dtype, causal, q, k, v, o, BH, S, D, err,
                   static_cast<cudaStream_t>(stream));
}

int kpb_attention(int variant, int dtype, const void* q, const void* k, const void* v, void* o,
                  int64_t BH, int64_t S, int64_t D, void* stream) {
  return attention_entry("attention", false, variant, dtype, q, k, v, o, BH, S, D, stream);
}

int kpb_attention_causal(int variant, int dtype, const void* q, const void* k, const void* v,
                         void* o, int64_t BH, int64_t S, int64_t D, void* stream) {
  return attention_entry("attention_causal", true, variant, dtype, q, k, v, o, BH, S, D, stream);
}

int kpb_qk_norm_rope(int variant, int dtype, const void* q, const void* k, const void* q_weight,
                     const void* k_weight, const float* cos_sin, const int64_t* positions,
                     void* q_out, void* k_out, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                     int64_t rot, int64_t max_pos, int64_t q_stride, int64_t k_stride, float eps,
                     int interleaved, void* stream) {
  g_last_error.clear();
  if (int rc = check_common("qk_norm_rope", variant, dtype)) return rc;
  if (int rc = check_rope("qk_norm_rope", T, Hq, Hkv, D, rot, max_pos)) return rc;
  if (T == 0 || Hq + Hkv == 0) return KPB_OK;
  if (positions == nullptr || (rot > 0 && max_pos > 0 && cos_sin == nullptr) ||
      (Hq > 0 && (!q || !q_weight || !q_out)) || (Hkv > 0 && (!k || !k_weight || !k_out)))
    return fail(KPB_EINVAL, "qk_norm_rope: null pointer");
  const size_t es = elem_bytes(dtype);
  if (off_by(q, es) || off_by(k, es) || off_by(q_weight, es) || off_by(k_weight, es) ||
      off_by(q_out, es) || off_by(k_out, es) || off_by(cos_sin, 4) || off_by(positions, 8))
    return fail(KPB_EINVAL, "qk_norm_rope: tensors must be element-aligned");
  unsigned* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return qk_norm_rope(variant, dtype, q, k, q_weight, k_weight, cos_sin, positions, q_out, k_out,
                      T, Hq, Hkv, D, rot, max_pos, q_stride, k_stride, eps, interleaved != 0, err,
                      static_cast<cudaStream_t>(stream));
}

size_t kpb_qk_norm_rope_backward_workspace_bytes(int64_t T, int64_t Hq, int64_t Hkv, int64_t D) {
  if (check_rope("qk_norm_rope_backward", T, Hq, Hkv, D, 0, 0) != KPB_OK) return 0;
  return qk_norm_rope_backward_workspace_bytes(T, Hq, Hkv, D);
}

int kpb_qk_norm_rope_backward(int variant, int dtype, const void* grad_q, const void* grad_k,
                              const void* q, const void* k, const void* q_weight,
                              const void* k_weight, const float* cos_sin,
                              const int64_t* positions, void* dq, void* dk, void* dq_weight,
                              void* dk_weight, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                              int64_t rot, int64_t max_pos, int64_t grad_q_stride,
                              int64_t grad_k_stride, int64_t q_stride, int64_t k_stride,
                              float eps, int interleaved, void* workspace,
                              size_t workspace_bytes, void* stream) {
  g_last_error.clear();
  const char* op = "qk_norm_rope_backward";
  if (int rc = check_common(op, variant, dtype)) return rc;
  if (int rc = check_rope(op, T, Hq, Hkv, D, rot, max_pos)) return rc;
  const std::string name(op);
  if (!dq_weight || !dk_weight || (T > 0 && !positions) ||
      (T > 0 && rot > 0 && max_pos > 0 && cos_sin == nullptr) ||
      (T * Hq > 0 && (!grad_q || !q || !q_weight || !dq)) ||
      (T * Hkv > 0 && (!grad_k || !k || !k_weight || !dk)))
    return fail(KPB_EINVAL, name + ": null pointer");
  const size_t es = elem_bytes(dtype);
  const void* ptrs[10] = {grad_q, grad_k, q, k, q_weight, k_weight, dq, dk, dq_weight, dk_weight};
  for (const void* p : ptrs)
    if (off_by(p, es)) return fail(KPB_EINVAL, name + ": tensors must be element-aligned");
  if (off_by(cos_sin, 4) || off_by(positions, 8))
    return fail(KPB_EINVAL, name + ": tensors must be element-aligned");
  const size_t need = qk_norm_rope_backward_workspace_bytes(T, Hq, Hkv, D);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(KPB_EINVAL, name + ": workspace too small (" + std::to_string(workspace_bytes) +
                                " bytes, need " + std::to_string(need) + ")");
  if (off_by(workspace, 16)) return fail(KPB_EINVAL, name + ": workspace must be 16-byte aligned");
  unsigned* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return qk_norm_rope_backward(variant, dtype, grad_q, grad_k, q, k, q_weight, k_weight, cos_sin,
                               positions, dq, dk, dq_weight, dk_weight, T, Hq, Hkv, D, rot,
                               max_pos, grad_q_stride, grad_k_stride, q_stride, k_stride, eps,
                               interleaved != 0, workspace, err,
                               static_cast<cudaStream_t>(stream));
}

int kpb_kv_cache_write(int variant, int dtype, int cache_dtype, const void* k, const void* v,
                       const int64_t* slots, void* k_cache, void* v_cache, float* k_scale,
                       float* v_scale, int64_t T, int64_t Hkv, int64_t D, int64_t num_pages,
                       int64_t page_size, int64_t k_stride, int64_t v_stride,
                       int64_t page_stride, void* stream) {
  g_last_error.clear();
  const char* op = "kv_cache_write";
  const KvLayout lay{num_pages, page_size, Hkv, D, page_stride};
  if (int rc = check_common(op, variant, dtype)) return rc;
  if (int rc = check_cache(op, dtype, cache_dtype, k_cache, v_cache, k_scale, v_scale, lay))
    return rc;
  if (!size_ok(T) || !size_ok(T * Hkv))
    return fail(KPB_EINVAL, "kv_cache_write: T and T * Hkv must be in [0, 2^31)");
  if (T == 0 || Hkv == 0) return KPB_OK;
  if (!k || !v || !slots) return fail(KPB_EINVAL, "kv_cache_write: null pointer");
  if (num_pages > 0 && k_cache == v_cache)
    return fail(KPB_EINVAL, "kv_cache_write: k_cache and v_cache must differ");
  if (num_pages > 0 && cache_dtype == KPB_E4M3 && k_scale == v_scale)
    return fail(KPB_EINVAL, "kv_cache_write: k_scale and v_scale must differ");
  if (off_by(k, elem_bytes(dtype)) || off_by(v, elem_bytes(dtype)) || off_by(slots, 8))
    return fail(KPB_EINVAL, "kv_cache_write: tensors must be element-aligned");
  unsigned* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return kv_cache_write(variant, dtype, cache_dtype, k, v, slots, k_cache, v_cache, k_scale,
                        v_scale, T, k_stride, v_stride, lay, err,
                        static_cast<cudaStream_t>(stream));
}

int kpb_kv_cache_read(int variant, int dtype, int cache_dtype, const void* k_cache,
                      const void* v_cache, const int64_t* slots, const float* k_scale,
                      const float* v_scale, void* k, void* v, int64_t T, int64_t Hkv, int64_t D,
                      int64_t num_pages, int64_t page_size, int64_t page_stride, void* stream) {
  g_last_error.clear();
  const char* op = "kv_cache_read";
  const KvLayout lay{num_pages, page_size, Hkv, D, page_stride};
  if (int rc = check_common(op, variant, dtype)) return rc;
  if (int rc = check_cache(op, dtype, cache_dtype, k_cache, v_cache, k_scale, v_scale, lay))
    return rc;
  if (!size_ok(T) || !size_ok(T * Hkv))
    return fail(KPB_EINVAL, "kv_cache_read: T and T * Hkv must be in [0, 2^31)");
  if (T == 0 || Hkv == 0) return KPB_OK;
  if (!k || !v || !slots) return fail(KPB_EINVAL, "kv_cache_read: null pointer");
  if (off_by(k, elem_bytes(dtype)) || off_by(v, elem_bytes(dtype)) || off_by(slots, 8))
    return fail(KPB_EINVAL, "kv_cache_read: tensors must be element-aligned");
  unsigned* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return kv_cache_read(variant, dtype, cache_dtype, k_cache, v_cache, slots, k_scale, v_scale, k,
                       v, T, lay, err, static_cast<cudaStream_t>(stream));
}

static int check_paged(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
  const std::string op("paged_attention");
  if (!size_ok(B) || !size_ok(Hq) || !size_ok(Hkv) || !size_ok(B * Hq))
    return fail(KPB_EINVAL, op + ": B, heads and B * Hq must be in [0, 2^31)");
  if (Hq > 0 && (Hkv == 0 || Hq % Hkv != 0))
    return fail(KPB_EINVAL, op + ": Hq must be a multiple of Hkv");
  if (D < 1 || D > kMaxHeadDim) return fail(KPB_EINVAL, op + ": D must be in [1, 256]");
  return KPB_OK;
}

size_t kpb_paged_attention_workspace_bytes(int variant, int64_t B, int64_t Hq, int64_t Hkv,
                                           int64_t D, int64_t max_len) {
  if (variant < 0 || variant >= kpb_num_variants("paged_attention") || !size_ok(max_len) ||
      check_paged(B, Hq, Hkv, D) != KPB_OK || B == 0 || Hq == 0)
    return 0;
  return paged_attention_workspace_bytes(variant, B, Hq, Hkv, D, max_len);
}

int kpb_paged_attention(int variant, int dtype, int cache_dtype, const void* q,
                        const void* k_cache, const void* v_cache, const int* block_table,
                        const int* seq_lens, const float* k_scale, const float* v_scale, void* o,
                        int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t num_pages,
                        int64_t page_size, int64_t max_pages, int64_t q_stride,
                        int64_t page_stride, int64_t table_stride, float scale, void* workspace,
                        size_t workspace_bytes, void* stream) {
  g_last_error.clear();
  const char* op = "paged_attention";
  const std::string name(op);
  const KvLayout lay{num_pages, page_size, Hkv, D, page_stride};
  if (int rc = check_common(op, variant, dtype)) return rc;
  if (int rc = check_cache(op, dtype, cache_dtype, k_cache, v_cache, k_scale, v_scale, lay))
    return rc;
  if (int rc = check_paged(B, Hq, Hkv, D)) return rc;
  if (!size_ok(max_pages) || !size_ok(max_pages * page_size))
    return fail(KPB_EINVAL, name + ": max_pages * page_size must be in [0, 2^31)");
  if (B == 0 || Hq == 0) return KPB_OK;
  if (!q || !seq_lens || !o || (max_pages > 0 && !block_table))
    return fail(KPB_EINVAL, name + ": null pointer");
  if (off_by(q, elem_bytes(dtype)) || off_by(o, elem_bytes(dtype)) || off_by(block_table, 4) ||
      off_by(seq_lens, 4))
    return fail(KPB_EINVAL, name + ": tensors must be element-aligned");
  const size_t need =
      paged_attention_workspace_bytes(variant, B, Hq, Hkv, D, max_pages * page_size);
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need)
      return fail(KPB_EINVAL, name + ": workspace too small (" + std::to_string(workspace_bytes) +
                                  " bytes, need " + std::to_string(need) + ")");
    if (off_by(workspace, 16))
      return fail(KPB_EINVAL, name + ": workspace must be 16-byte aligned");
  }
  unsigned* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  return paged_attention(variant, dtype, cache_dtype, q, k_cache, v_cache, block_table, seq_lens,
                         k_scale, v_scale, o, B, Hq, max_pages, q_stride, table_stride, scale,
                         lay, workspace, workspace_bytes, err, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
