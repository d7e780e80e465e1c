// qserve.cu — C ABI of the ends of a serving step (declared in
// include/qlinear.h): page tables and slots from request lengths, and drawing
// tokens from logits.  Argument checks, launch shapes and launches; every
// entry point returns a status and allocates nothing.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "../../include/qlinear.h"
#include "ql_host.h"
#include "qplan.cuh"
#include "qsample.cuh"

namespace {

constexpr int kMaxDevices = 64;

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// One cluster of `cluster` CTAs along x after another.
template <typename Kern, typename... Args>
int launch_clusters(Kern kernel, unsigned ctas, unsigned cluster, unsigned threads, size_t smem, void* stream,
                    int64_t flags, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (flags & QL_FLAG_PDL) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return QL_ERR_CUDA;
  }
  return QL_OK;
}

// Lets a kernel use `smem` bytes and clusters of 16, once per device.
template <typename Kern>
int allow(Kern kernel, size_t smem, std::atomic<unsigned char>* done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    return QL_ERR_DEVICE;
  }
  if (done[dev].load(std::memory_order_acquire)) return QL_OK;
  if ((smem > 0 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    cudaGetLastError();
    return QL_ERR_CUDA;
  }
  done[dev].store(1, std::memory_order_release);
  return QL_OK;
}

constexpr int64_t kFewRequests = 1024, kFewTokens = 2048;

// ------------------------------------------------------------------- sampling
template <typename T>
int run_sample(const ql::smp::Params& p, bool few, int sms, void* stream, int64_t flags) {
  using namespace ql::smp;
  auto kernel = sample_kernel<T>;
  static std::atomic<unsigned char> done[kMaxDevices];
  const int st = allow(kernel, kStaged, done);
  if (st != QL_OK) return st;
  const int64_t runs = cdiv(p.vocab, Type<T>::kLanes);
  auto passes = [&](int ctas) { return cdiv(cdiv(runs, ctas), kThreads); };
  // As many CTAs a row as the SMs have places for (two on each), and fewer of the larger clusters, which find their places
  // less easily.  151936 logits, fp16, device us by CTAs a row 1 | 2 | 4 | 8 | 16:
  //   top-k 50, top-p 0.95:   1 row  20 | 16 | 14 | 13 | 12     16 rows 23 | 18 | 17 | 16 | 27     64 rows 26 | 22 | 20 | 33 | 74
  //   all of them:            1 row  26 | 17 | 12 |  9 |  8     16 rows 62 | 37 | 25 | 18 | 18     64 rows 83 | 54 | 37 | 35 | 53
  //                         128 rows 97 | 62 | 56 | 61 |  98   256 rows 120 | 86 | 89 | 114 | 192
  //   top-p 0.9:              1 row 156 | 95 | 64 | 44 | 40     64 rows 224 | 143 | 104 | 124 | 226   256 rows 298 | 300 | 346 | 459 | 845
  // fp32 and smaller vocabularies, as the rule has it | the best:
  //   151936 fp32, top-p 0.9: 1 row 42 | 42   64 rows 116 | 116  128 rows 198 | 197  256 rows 350 | 350
  //     all of them:                          64 rows  43 | 42   128 rows  72 | 61   256 rows 109 | 100
  //    32003 fp16, top-p 0.9: 1 row 33 | 33   64 rows  48 | 48   128 rows  61 | 61   256 rows 110 | 85
  //    32003 fp32, top-p 0.9: 1 row 34 | 31   64 rows  49 | 49   128 rows  64 | 64   256 rows 118 | 106
  //     4099 fp16, top-p 0.9: 1 row 15 | 14   64 rows  37 | 37   128 rows  39 | 39   256 rows  55 | 44
  // Where all rows are known to keep few, one CTA is less to start and to meet:
  //   top-k 50, top-p 0.95: 128 rows 34 | 25 | 40     256 rows 39 | 48 | 75        the largest: 128 rows 15 | 12     256 rows 18 | 22
  auto room = [&](int ctas) { return ctas <= 2 ? (few ? 2 : 4) * sms : ctas <= 4 ? 2 * sms : ctas <= 8 ? sms : sms / 2; };
  int ctas = 1;
  while (ctas < kMaxCtas && passes(ctas) > 1 && ((int64_t)p.rows * 2 * ctas <= room(2 * ctas) || passes(ctas) * kWarps > kBlocks)) ctas *= 2;
  const size_t bytes = (size_t)passes(ctas) * kThreads * 16;
  const int staged = bytes <= kStaged;
  return launch_clusters(kernel, (unsigned)p.rows * ctas, (unsigned)ctas, kThreads, staged ? bytes : 0, stream, flags, p, staged);
}

}  // namespace

extern "C" {

int ql_plan_step(const ql_plan_step_args* a, void* stream) {
  if (!a) return QL_ERR_NULL_POINTER;
  if (a->batch < 0 || a->batch > ql::plan::kMaxBatch || a->table_width < 0 || a->num_pages < 0 ||
      a->num_pages > INT_MAX || a->max_tokens < 0 || a->max_tokens >= INT_MAX ||
      a->batch * std::min<int64_t>(a->table_width, INT_MAX) > INT_MAX)
    return QL_ERR_BAD_SHAPE;
  if (a->page_size < 1 || a->page_size > 65536 || (a->page_size & (a->page_size - 1)) != 0) return QL_ERR_UNSUPPORTED;
  if (a->table_stride < a->table_width) return QL_ERR_BAD_STRIDE;
  if (!a->cu_q || !a->refused || !a->free_count || (a->batch > 0 && (!a->lens || !a->fresh)) ||
      (a->batch > 0 && a->table_width > 0 && !a->page_table) || (a->num_pages > 0 && !a->free_pages) ||
      (a->max_tokens > 0 && (!a->slots || !a->positions)))
    return QL_ERR_NULL_POINTER;
  for (const void* p : {a->page_table, a->lens, a->free_pages, a->free_count, a->cu_q, a->refused})
    if (!aligned(p, 4)) return QL_ERR_UNSUPPORTED;
  if (!aligned(a->keep, 4) || !aligned(a->fresh, 4) || !aligned(a->slots, 16) || !aligned(a->positions, 16))
    return QL_ERR_UNSUPPORTED;
  ql_host::Device dev;
  int st = ql_host::current(&dev);
  if (st != QL_OK) return st;
  ql::plan::Params p = {};
  p.table = static_cast<int*>(a->page_table);
  p.lens = static_cast<int*>(a->lens);
  p.stack = static_cast<int*>(a->free_pages);
  p.count = static_cast<int*>(a->free_count);
  p.keep = static_cast<const int*>(a->keep);
  p.fresh = static_cast<const int*>(a->fresh);
  p.cu_q = static_cast<int*>(a->cu_q);
  p.slots = static_cast<long long*>(a->slots);
  p.positions = static_cast<int*>(a->positions);
  p.refused = static_cast<int*>(a->refused);
  p.table_stride = a->table_stride;
  p.max_tokens = a->max_tokens;
  p.batch = (int)a->batch;
  p.width = (int)std::min<int64_t>(a->table_width, INT_MAX);
  p.num_pages = (int)a->num_pages;
  p.page_shift = __builtin_ctzll((unsigned long long)a->page_size);
  auto kernel = ql::plan::plan_kernel;
  static std::atomic<unsigned char> done[kMaxDevices];
  if ((st = allow(kernel, (4 * (size_t)ql::plan::kMaxBatch + 2) * sizeof(int), done)) != QL_OK) return st;
  // One CTA for all requests as far as its threads go, else a cluster of 8, each of which scans them all.  More tokens than
  // its threads have in two rounds go to all SMs: each lookup is a search of log2(batch) steps in shared memory, of which
  // 6000 take one SM longer (6 us) than a launch.
  const bool few_requests = a->batch <= kFewRequests, few_tokens = a->max_tokens <= kFewTokens;
  p.tokens = few_tokens;
  const int64_t wanted = std::max(a->batch, few_tokens ? a->max_tokens : cdiv(a->max_tokens, a->page_size));
  const unsigned ctas = few_requests ? 1 : 8;
  const unsigned threads = (unsigned)std::min<int64_t>(std::max<int64_t>(cdiv(wanted, 32) * 32, 128), ql::plan::kThreads);
  st = launch_clusters(kernel, ctas, ctas, threads, (4 * (size_t)a->batch + 2) * sizeof(int), stream, a->flags, p);
  if (st != QL_OK || few_tokens) return st;
  return launch_clusters(ql::plan::token_kernel, (unsigned)cdiv(a->max_tokens, 4 * ql::plan::kTokenThreads), 1,
                         ql::plan::kTokenThreads, ((size_t)a->batch + 1) * sizeof(int), stream, a->flags, p);
}

int ql_sample_tokens(const ql_sample_tokens_args* a, void* stream) {
  if (!a) return QL_ERR_NULL_POINTER;
  if (a->rows < 0 || a->rows > INT_MAX / ql::smp::kMaxCtas || a->vocab < 1 || a->vocab > QL_SAMPLE_MAX_VOCAB)
    return QL_ERR_BAD_SHAPE;
  if (a->dtype != QL_DTYPE_F16 && a->dtype != QL_DTYPE_BF16 && a->dtype != QL_DTYPE_F32) return QL_ERR_UNSUPPORTED;
  const size_t bytes = a->dtype == QL_DTYPE_F32 ? 4 : 2;
  if (a->rows == 0) return QL_OK;
  if (!a->logits || !a->uniform || !a->ids) return QL_ERR_NULL_POINTER;
  if (a->row_stride < 0 || (a->rows > 1 && a->row_stride < a->vocab)) return QL_ERR_BAD_STRIDE;
  if (!aligned(a->logits, bytes) || !aligned(a->uniform, 4) || !aligned(a->temperature, 4) || !aligned(a->top_k, 4) ||
      !aligned(a->top_p, 4) || !aligned(a->min_p, 4) || !aligned(a->ids, 8) || !aligned(a->logprobs, 4))
    return QL_ERR_UNSUPPORTED;
  ql_host::Device dev;
  const int st = ql_host::current(&dev);
  if (st != QL_OK) return st;
  ql::smp::Params p = {};
  p.logits = a->logits;
  p.uniform = static_cast<const float*>(a->uniform);
  p.temperature = static_cast<const float*>(a->temperature);
  p.top_k = static_cast<const int*>(a->top_k);
  p.top_p = static_cast<const float*>(a->top_p);
  p.min_p = static_cast<const float*>(a->min_p);
  p.ids = static_cast<long long*>(a->ids);
  p.logprobs = static_cast<float*>(a->logprobs);
  p.temperature_all = a->temperature_all;
  p.top_k_all = a->top_k_all;
  p.top_p_all = a->top_p_all;
  p.min_p_all = a->min_p_all;
  p.stride = a->row_stride;
  p.rows = (int)a->rows;
  p.vocab = (int)a->vocab;
  p.vec = aligned(a->logits, 16) && (a->rows == 1 || a->row_stride * (int64_t)bytes % 16 == 0);
  const bool few = (!a->temperature && !(a->temperature_all > 0.0)) || (!a->top_k && a->top_k_all > 0 && a->top_k_all <= ql::smp::kFew / 2);
  switch (a->dtype) {
    case QL_DTYPE_F16: return run_sample<__half>(p, few, dev.sms, stream, a->flags);
    case QL_DTYPE_BF16: return run_sample<__nv_bfloat16>(p, few, dev.sms, stream, a->flags);
    default: return run_sample<float>(p, few, dev.sms, stream, a->flags);
  }
}

}  // extern "C"
