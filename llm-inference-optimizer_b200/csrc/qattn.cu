// qattn.cu — C ABI of the attention side of libqlinear.so (declared in
// include/qlinear.h): rotary positions, the quantised paged cache and
// attention over it.  Argument checks, variant choice and launches; every
// entry point returns a status and allocates nothing.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>

#include "../../include/qlinear.h"
#include "ql_host.h"
#include "qattend.cuh"
#include "qcache.cuh"
#include "qtree.cuh"

namespace {

using ql::kvc::Pool;
using ql::kvc::Rows;
using ql::kvc::Turn;

constexpr int kMaxDevices = 64;

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename Kern, typename... Args>
int launch(Kern kernel, dim3 grid, dim3 block, size_t smem, void* stream, int64_t flags, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = (flags & QL_FLAG_PDL) ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return QL_ERR_CUDA;
  }
  return QL_OK;
}

bool act_dtype(int64_t d) { return d == QL_DTYPE_F16 || d == QL_DTYPE_BF16; }
bool index_bytes(int64_t n) { return n == 4 || n == 8; }

// A [tokens][heads][head_dim] tensor of 16-bit elements.
int make_rows(Rows* r, const void* p, int64_t token_stride, int64_t head_stride, int64_t head_dim) {
  if (!p) return QL_ERR_NULL_POINTER;
  if (!aligned(p, 2)) return QL_ERR_UNSUPPORTED;
  if (token_stride < 0 || head_stride < 0) return QL_ERR_BAD_STRIDE;
  r->p = p;
  r->token_stride = token_stride;
  r->head_stride = head_stride;
  r->vec = aligned(p, 16) && token_stride % 8 == 0 && head_stride % 8 == 0 && head_dim % 8 == 0;
  return QL_OK;
}

int make_turn(Turn* t, const void* table, const void* positions, int64_t position_bytes, int64_t max_positions,
              int64_t rotary_dim, int64_t head_dim, int64_t layout, int64_t inverse) {
  if (rotary_dim <= 0 || rotary_dim % 8 != 0 || rotary_dim > head_dim || max_positions <= 0)
    return QL_ERR_BAD_SHAPE;
  if (!table || !positions) return QL_ERR_NULL_POINTER;
  if (!index_bytes(position_bytes) || !aligned(table, 16) || !aligned(positions, (size_t)position_bytes) ||
      (layout != QL_ROTARY_HALF && layout != QL_ROTARY_INTERLEAVED))
    return QL_ERR_UNSUPPORTED;
  t->table = static_cast<const float2*>(table);
  t->positions = positions;
  t->max_positions = max_positions;
  t->wide = position_bytes == 8;
  t->rotary_dim = (int)rotary_dim;
  t->interleaved = layout == QL_ROTARY_INTERLEAVED;
  t->inverse = inverse != 0;
  return QL_OK;
}

int make_pool(Pool* c, const ql_kv_cache& a) {
  if (!a.k_codes || !a.k_scales || !a.v_codes || !a.v_scales) return QL_ERR_NULL_POINTER;
  if (a.bits != 8 && a.bits != 4) return QL_ERR_UNSUPPORTED;
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return QL_ERR_UNSUPPORTED;
  if (a.page_size < 16 || a.page_size > 65536 || (a.page_size & (a.page_size - 1)) != 0) return QL_ERR_UNSUPPORTED;
  if (a.num_pages <= 0 || a.kv_heads <= 0 || a.num_pages > INT_MAX || a.kv_heads > 65536 ||
      a.kv_heads * a.page_size > INT_MAX)
    return QL_ERR_BAD_SHAPE;
  const int64_t row = a.head_dim * a.bits / 8, groups = a.bits == 8 ? 1 : a.head_dim / ql::kvc::kGroup4;
  const int64_t rows = a.kv_heads * a.page_size;
  if (a.k_page_stride < rows * row || a.v_page_stride < rows * row || a.k_scale_page_stride < rows * groups ||
      a.v_scale_page_stride < rows * groups)
    return QL_ERR_BAD_STRIDE;
  if (std::max(a.k_page_stride, a.v_page_stride) > UINT_MAX || std::max(a.k_scale_page_stride, a.v_scale_page_stride) > UINT_MAX)
    return QL_ERR_UNSUPPORTED;
  // rows are read and written in 16-byte words
  if (!aligned(a.k_codes, 16) || !aligned(a.v_codes, 16) || !aligned(a.k_scales, 16) || !aligned(a.v_scales, 16) ||
      a.k_page_stride % 16 || a.v_page_stride % 16 || a.k_scale_page_stride % 8 || a.v_scale_page_stride % 8)
    return QL_ERR_UNSUPPORTED;
  c->k_codes = static_cast<unsigned char*>(a.k_codes);
  c->v_codes = static_cast<unsigned char*>(a.v_codes);
  c->k_scales = static_cast<unsigned short*>(a.k_scales);
  c->v_scales = static_cast<unsigned short*>(a.v_scales);
  c->k_page = (unsigned)a.k_page_stride;
  c->v_page = (unsigned)a.v_page_stride;
  c->ks_page = (unsigned)a.k_scale_page_stride;
  c->vs_page = (unsigned)a.v_scale_page_stride;
  c->slots = a.num_pages * a.page_size;
  c->page_shift = __builtin_ctzll((unsigned long long)a.page_size);
  c->heads = (int)a.kv_heads;
  c->row_bytes = (int)row;
  c->groups = (int)groups;
  c->bits = (int)a.bits;
  return QL_OK;
}

// Raise the dynamic shared-memory limit of a kernel once per device.
template <typename Kern>
int allow_smem(Kern kernel, size_t bytes, std::atomic<unsigned char>* done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    return QL_ERR_DEVICE;
  }
  if (done[dev].load(std::memory_order_acquire)) return QL_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) {
    cudaGetLastError();
    return QL_ERR_CUDA;
  }
  done[dev].store(1, std::memory_order_release);
  return QL_OK;
}

ql::kvc::Divisor divisor(int64_t d) {
  unsigned log = 0;
  while ((1ll << log) < d) ++log;
  return {(unsigned)cdiv(1ll << (31 + log), d), 31 + log};
}

// Threads over tokens and `per_thread` heads each; with few tokens a head
// each, since then all is latency.
ql::kvc::Grid make_grid(int64_t tokens, int64_t heads, int64_t chunks, int per_thread, int sms) {
  ql::kvc::Grid g;
  const int64_t wanted = tokens <= sms ? heads : cdiv(heads, per_thread);
  g.chunks = (int)chunks;
  g.beside = (int)std::max<int64_t>(1, std::min(wanted, 256 / chunks));
  const int64_t threads = g.beside * chunks;
  g.tokens = tokens <= sms ? 1 : (int)(256 / threads);
  g.by_token = divisor(threads);
  g.by_chunks = divisor(chunks);
  return g;
}
unsigned threads_of(const ql::kvc::Grid& g) { return (unsigned)cdiv((int64_t)g.beside * g.chunks * g.tokens, 32) * 32; }

template <typename T, int LANES>
int run_append_bits(const ql::kvc::AppendParams& p, dim3 grid, dim3 block, void* stream, int64_t flags) {
  return p.cache.bits == 8 ? launch(ql::kvc::append_kernel<T, LANES, 8>, grid, block, 0, stream, flags, p)
                           : launch(ql::kvc::append_kernel<T, LANES, 4>, grid, block, 0, stream, flags, p);
}

template <typename T>
int run_append(ql::kvc::AppendParams p, int64_t chunks, int sms, void* stream, int64_t flags) {
  p.grid = make_grid(p.tokens, p.cache.heads, chunks, 1, sms);
  p.kv_ctas = (int)cdiv(p.tokens, p.grid.tokens);
  unsigned threads = threads_of(p.grid);
  int64_t ctas = p.kv_ctas;
  if (p.q.heads > 0) {
    p.q.grid = make_grid(p.tokens, p.q.heads, chunks, ql::kvc::kHeads, sms);
    threads = std::max(threads, threads_of(p.q.grid));
    ctas += cdiv(p.tokens, p.q.grid.tokens);
  }
  if (ctas > INT_MAX) return QL_ERR_BAD_SHAPE;
  const dim3 grid((unsigned)ctas), block(threads);
  switch (chunks) {
    case 8: return run_append_bits<T, 8>(p, grid, block, stream, flags);
    case 16: return run_append_bits<T, 16>(p, grid, block, stream, flags);
    default: return run_append_bits<T, 32>(p, grid, block, stream, flags);
  }
}

// The tensor-core kernel (head_dim 64 and 128; 256 does not fit its memories)
// is taken above kTreeRows rows of a request under one key/value head, where
// the streaming kernel would have kTreeWork units of work a CTA and more: units
// of 128 keys by 16 rows, an item's start and end counted as kItemWork of them.
// Below, the tensor-core kernel's start and end (22 us) outweigh its rate.
// 32 heads over 4 of 128, 8 bits, fp16 / bf16, us, streaming | tensor-core:
//   8 requests of up to 6001, 64 rows:    45 / 47 | 45 / 54
//                            128 rows:    75 / 78 | 47 / 56
//   16 requests of up to 600, 72 rows:    33 / 35 | 23 / 28    (28 units)
//   1 request of 16001,      128 rows:    46 / 48 | 44 / 49    (29 units)
//   2 requests of up to 3001, 256 rows:   34 / 35 | 38 / 44    (27.7 units)
//   4 requests of up to 1500, 128 rows:   25 / 26 | 26 / 31    (17 units)
//   1 request of 600,        512 rows:    22 / 23 | 30 / 35    (11 units)
// That is of requests alike.  A batch of few trees among single tokens has the
// rows of its mean, not of its largest, and 256 rows for every single token cost
// the tensor-core kernel more than they save: it is taken above kMeanRows rows
// a request on average.  64 requests of up to 8000, 8 bits, fp16, us, streaming | tensor-core:
//   28 heads over 4, 1 token each:                   7 rows:   71 | 201
//                    one tree of 64, 63 tokens:     14 rows:  148 | 237
//                    4 tokens each:                 28 rows:  194 | 219
//                    4 trees of 64, 60 tokens:      35 rows:  291 | 253    (up to 2000: 109 | 118)
//                    32 trees of 16, 32 tokens:     60 rows:  399 | 214
//   32 heads over 8, 4 trees of 64, 60 tokens:      20 rows:  402 | 454
//                    16 trees of 64, 48 tokens:     67 rows: 1001 | 465
// The same mean tells how many rows the streaming kernel takes at once (32 heads over 8, one tree of 64 and 63
// tokens, 8 rows: 193 us with tiles of 8, 238 with tiles of 16).
constexpr int64_t kTreeRows = 64, kMeanRows = 32, kTreeWork = 28, kItemWork = 8;

struct Attention {
  ql::att::Params p;
  int64_t max_q, max_kv, flags;
  int64_t max_rows, mean_rows;   // of a request under one key/value head
  void* workspace;
  size_t workspace_bytes;
  void* stream;
  int sms;
};

template <int D, int BITS, int NT>
size_t stream_workspace(int sms) {
  using S = ql::att::Shape<D, BITS, NT>;
  const size_t ctas = std::min(ql::att::kMaxCtas, S::kCtas * sms);
  return ql::att::kHeaderBytes + 2 * ctas * S::kPartial * sizeof(float);
}

template <typename T, int D, int BITS, int NT>
int run_stream(const Attention& a) {
  using S = ql::att::Shape<D, BITS, NT>;
  if (a.workspace_bytes < stream_workspace<D, BITS, NT>(a.sms)) return QL_ERR_WORKSPACE;
  auto kernel = ql::att::stream_kernel<T, D, BITS, NT>;
  static std::atomic<unsigned char> done[kMaxDevices];
  const int st = allow_smem(kernel, S::kSmem, done);
  if (st != QL_OK) return st;
  // as many CTAs as the SMs hold at once, and no more than the bounds on the work can use
  const int64_t tiles = cdiv(std::max<int64_t>(a.max_q, 1) * a.p.group, S::kRows);
  const int64_t runs = cdiv(std::max<int64_t>(a.max_kv, 1), ql::att::kUnitKeys * ql::att::kMinUnits);
  int64_t ctas = std::min<int64_t>(ql::att::kMaxCtas, (int64_t)S::kCtas * a.sms);
  const double bound = (double)a.p.batch * a.p.cache.heads * (double)tiles * (double)runs;
  if (bound < (double)ctas) ctas = std::max<int64_t>((int64_t)bound, 1);
  return launch(kernel, dim3((unsigned)ctas), dim3(ql::att::kThreads), S::kSmem, a.stream, a.flags, a.p,
                static_cast<unsigned*>(a.workspace),
                reinterpret_cast<float*>(static_cast<char*>(a.workspace) + ql::att::kHeaderBytes));
}

template <int D, int BITS>
size_t tree_workspace(int sms) {
  return ql::att::kHeaderBytes + 2 * (size_t)std::min(ql::att::kMaxCtas, sms) * ql::tree::Shape<D, BITS>::kPartial * sizeof(float);
}

template <typename T, int D, int BITS>
int run_tree(const Attention& a) {
  using S = ql::tree::Shape<D, BITS>;
  if (a.workspace_bytes < tree_workspace<D, BITS>(a.sms)) return QL_ERR_WORKSPACE;
  auto kernel = ql::tree::tree_kernel<T, D, BITS>;
  static std::atomic<unsigned char> done[kMaxDevices];
  const int st = allow_smem(kernel, S::kSmem, done);
  if (st != QL_OK) return st;
  const int64_t tiles = cdiv(std::max<int64_t>(a.max_q, 1) * a.p.group, ql::tree::kRows);
  const int64_t runs = cdiv(std::max<int64_t>(a.max_kv, 1), ql::att::kUnitKeys * ql::tree::kMinUnits);
  int64_t ctas = std::min<int64_t>(ql::att::kMaxCtas, a.sms);
  const double bound = (double)a.p.batch * a.p.cache.heads * (double)tiles * (double)runs;
  if (bound < (double)ctas) ctas = std::max<int64_t>((int64_t)bound, 1);
  return launch(kernel, dim3((unsigned)ctas), dim3(ql::tree::kThreads), S::kSmem, a.stream, a.flags, a.p,
                static_cast<unsigned*>(a.workspace),
                reinterpret_cast<float*>(static_cast<char*>(a.workspace) + ql::att::kHeaderBytes));
}

template <typename T, int D, int BITS>
int run_rows(const Attention& a) {
  if constexpr (D <= 128) {
    const int64_t units = cdiv(a.max_kv, ql::att::kUnitKeys) + kItemWork;
    const double work = (double)a.p.batch * a.p.cache.heads * (double)cdiv(a.max_rows, 16) * (double)units;
    const bool tree = a.max_rows > kTreeRows && a.mean_rows > kMeanRows && work >= (double)(kTreeWork * a.sms);
    if (!(a.flags & QL_FLAG_FORCE_GEMV) && (tree || (a.flags & QL_FLAG_FORCE_GEMM))) return run_tree<T, D, BITS>(a);
  }
  return a.mean_rows <= 8 ? run_stream<T, D, BITS, 1>(a) : run_stream<T, D, BITS, 2>(a);
}

template <typename T>
int run_attention(const Attention& a, int64_t head_dim) {
  const bool eight = a.p.cache.bits == 8;
  switch (head_dim) {
    case 64: return eight ? run_rows<T, 64, 8>(a) : run_rows<T, 64, 4>(a);
    case 128: return eight ? run_rows<T, 128, 8>(a) : run_rows<T, 128, 4>(a);
    default: return eight ? run_rows<T, 256, 8>(a) : run_rows<T, 256, 4>(a);
  }
}

}  // namespace

extern "C" {

int ql_rotary(const ql_rotary_args* a, void* stream) {
  if (!a) return QL_ERR_NULL_POINTER;
  if (a->tokens < 0 || a->heads < 0 || a->tokens > INT_MAX || a->head_dim <= 0 || a->head_dim % 8 != 0 ||
      a->head_dim > 2048 || a->heads > 65536 || a->heads * a->head_dim > INT_MAX)
    return QL_ERR_BAD_SHAPE;
  if (!act_dtype(a->dtype)) return QL_ERR_UNSUPPORTED;
  if (a->tokens == 0 || a->heads == 0) return QL_OK;
  ql::kvc::RotaryParams p = {};
  int st = make_rows(&p.x, a->x, a->x_token_stride, a->x_head_stride, a->head_dim);
  if (st == QL_OK) st = make_rows(&p.out, a->out, a->out_token_stride, a->out_head_stride, a->head_dim);
  if (st == QL_OK)
    st = make_turn(&p.turn, a->table, a->positions, a->position_bytes, a->max_positions, a->rotary_dim, a->head_dim,
                   a->layout, a->inverse);
  if (st != QL_OK) return st;
  ql_host::Device dev;
  if ((st = ql_host::current(&dev)) != QL_OK) return st;
  p.tokens = (int)a->tokens;
  p.heads = (int)a->heads;
  p.grid = make_grid(a->tokens, a->heads, a->head_dim / 8, ql::kvc::kHeads, dev.sms);
  p.err = dev.err_word;
  const dim3 grid((unsigned)cdiv(a->tokens, p.grid.tokens)), block(threads_of(p.grid));
  return a->dtype == QL_DTYPE_F16 ? launch(ql::kvc::rotary_kernel<__half>, grid, block, 0, stream, a->flags, p)
                                  : launch(ql::kvc::rotary_kernel<__nv_bfloat16>, grid, block, 0, stream, a->flags, p);
}

int ql_kv_append(const ql_kv_append_args* a, void* stream) {
  if (!a) return QL_ERR_NULL_POINTER;
  if (a->tokens < 0 || a->tokens > INT_MAX || a->q_heads < 0 || a->q_heads > 65536) return QL_ERR_BAD_SHAPE;
  if (!act_dtype(a->dtype) || !index_bytes(a->slot_bytes)) return QL_ERR_UNSUPPORTED;
  ql::kvc::AppendParams p = {};
  int st = make_pool(&p.cache, a->cache);
  if (st != QL_OK) return st;
  if (a->tokens == 0) return QL_OK;
  const int64_t d = a->cache.head_dim;
  if (!a->slots) return QL_ERR_NULL_POINTER;
  if (!aligned(a->slots, (size_t)a->slot_bytes)) return QL_ERR_UNSUPPORTED;
  if ((st = make_rows(&p.k, a->k, a->k_token_stride, a->k_head_stride, d)) != QL_OK) return st;
  if ((st = make_rows(&p.v, a->v, a->v_token_stride, a->v_head_stride, d)) != QL_OK) return st;
  if (a->q_heads > 0) {
    if ((st = make_rows(&p.q.x, a->q, a->q_token_stride, a->q_head_stride, d)) != QL_OK) return st;
    if ((st = make_rows(&p.q.out, a->q_out, a->q_out_token_stride, a->q_out_head_stride, d)) != QL_OK) return st;
    if (a->rotary_dim == 0) return QL_ERR_BAD_SHAPE;   // q is there to be turned: no angles, no positions
  }
  if (a->rotary_dim != 0) {
    st = make_turn(&p.q.turn, a->table, a->positions, a->position_bytes, a->max_positions, a->rotary_dim, d, a->layout,
                   0);
    if (st != QL_OK) return st;
  }
  ql_host::Device dev;
  if ((st = ql_host::current(&dev)) != QL_OK) return st;
  p.slots = a->slots;
  p.wide_slots = a->slot_bytes == 8;
  p.tokens = p.q.tokens = (int)a->tokens;
  p.q.heads = (int)a->q_heads;
  p.q.err = dev.err_word;
  return a->dtype == QL_DTYPE_F16 ? run_append<__half>(p, d / 8, dev.sms, stream, a->flags)
                                  : run_append<__nv_bfloat16>(p, d / 8, dev.sms, stream, a->flags);
}

int ql_kv_read(const ql_kv_read_args* a, void* stream) {
  if (!a) return QL_ERR_NULL_POINTER;
  if (a->tokens < 0 || a->tokens > INT_MAX) return QL_ERR_BAD_SHAPE;
  if (!act_dtype(a->dtype) || !index_bytes(a->slot_bytes)) return QL_ERR_UNSUPPORTED;
  ql::kvc::ReadParams p = {};
  int st = make_pool(&p.cache, a->cache);
  if (st != QL_OK) return st;
  if (a->tokens == 0) return QL_OK;
  if (!a->slots || !a->k || !a->v) return QL_ERR_NULL_POINTER;
  if (!aligned(a->slots, (size_t)a->slot_bytes) || !aligned(a->k, 16) || !aligned(a->v, 16))
    return QL_ERR_UNSUPPORTED;
  // tokens side by side in a CTA, or CTAs to a token
  const int64_t per_token = a->cache.kv_heads * a->cache.head_dim / 8;
  const int side = per_token <= 256 ? (int)(256 / per_token) : 1, split = (int)cdiv(per_token, 256);
  const int64_t blocks = cdiv(a->tokens, (int64_t)side * ql::kvc::kTokens) * split;
  const int log_chunks = __builtin_ctzll((unsigned long long)a->cache.head_dim / 8);
  ql_host::Device dev;
  if ((st = ql_host::current(&dev)) != QL_OK) return st;
  p.slots = a->slots;
  p.wide_slots = a->slot_bytes == 8;
  p.tokens = a->tokens;
  p.k = a->k;
  p.v = a->v;
  p.err = dev.err_word;
  if (blocks > INT_MAX) return QL_ERR_BAD_SHAPE;
  const dim3 grid((unsigned)blocks), block(256);
  return a->dtype == QL_DTYPE_F16
             ? launch(ql::kvc::read_kernel<__half>, grid, block, 0, stream, a->flags, p, log_chunks, side, split)
             : launch(ql::kvc::read_kernel<__nv_bfloat16>, grid, block, 0, stream, a->flags, p, log_chunks, side, split);
}

int ql_tree_attention(const ql_tree_attention_args* a, void* stream) {
  if (!a) return QL_ERR_NULL_POINTER;
  if (a->batch < 0 || a->total_q < 0 || a->batch > 65535 || a->total_q > INT_MAX || a->q_heads < 0 ||
      a->q_heads > 65536 || a->table_width < 0 || a->table_width > INT_MAX || a->mask_words < 0 ||
      a->mask_words > 1024)
    return QL_ERR_BAD_SHAPE;
  if (!act_dtype(a->dtype)) return QL_ERR_UNSUPPORTED;
  ql::att::Params p = {};
  int st = make_pool(&p.cache, a->cache);
  if (st != QL_OK) return st;
  if (a->q_heads % a->cache.kv_heads != 0 || a->total_q * a->q_heads > INT_MAX) return QL_ERR_BAD_SHAPE;
  if (a->batch == 0 || a->total_q == 0 || a->q_heads == 0) return QL_OK;
  if (!a->cu_q && a->total_q % a->batch != 0) return QL_ERR_BAD_SHAPE;
  if (!a->out || !a->kv_lens || !a->workspace || (!a->page_table && a->table_width > 0)) return QL_ERR_NULL_POINTER;
  if ((st = make_rows(&p.q, a->q, a->q_token_stride, a->q_head_stride, a->cache.head_dim)) != QL_OK) return st;
  if (a->table_stride < a->table_width) return QL_ERR_BAD_STRIDE;
  if (!aligned(a->out, 16) || !aligned(a->lse, 4) || !aligned(a->page_table, 4) || !aligned(a->kv_lens, 4) ||
      !aligned(a->cu_q, 4) || !aligned(a->mask, 8) || !aligned(a->workspace, 16))
    return QL_ERR_UNSUPPORTED;
  ql_host::Device dev;
  if ((st = ql_host::current(&dev)) != QL_OK) return st;
  p.out = a->out;
  p.lse = static_cast<float*>(a->lse);
  p.page_table = static_cast<const int*>(a->page_table);
  p.kv_lens = static_cast<const int*>(a->kv_lens);
  p.cu_q = static_cast<const int*>(a->cu_q);
  p.mask = static_cast<const unsigned long long*>(a->mask);
  p.table_stride = a->table_stride;
  p.table_width = (int)a->table_width;
  p.num_pages = (int)a->cache.num_pages;
  p.batch = (int)a->batch;
  p.total_q = (int)a->total_q;
  p.q_heads = (int)a->q_heads;
  p.group = (int)(a->q_heads / a->cache.kv_heads);
  p.by_group = divisor(p.group);
  p.mask_words = (int)a->mask_words;
  p.scale_log2 = (float)(a->scale * 1.4426950408889634);
  p.err = dev.err_word;
  // the caller's bounds, where total_q and the table do not give better ones
  const int64_t max_q = std::min(a->cu_q ? std::max<int64_t>(a->max_q, 1) : a->total_q / a->batch, a->total_q);
  const int64_t max_kv = std::min(std::max<int64_t>(a->max_kv, 1), a->table_width * a->cache.page_size);
  const Attention work = {p, max_q, max_kv, a->flags, max_q * p.group, cdiv(a->total_q * p.group, a->batch), a->workspace,
                          (size_t)std::max<int64_t>(a->workspace_bytes, 0), stream, dev.sms};
  return a->dtype == QL_DTYPE_F16 ? run_attention<__half>(work, a->cache.head_dim)
                                  : run_attention<__nv_bfloat16>(work, a->cache.head_dim);
}

uint64_t ql_capture_id(void* stream) {
  cudaStreamCaptureStatus status;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &id) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

size_t ql_tree_attention_workspace_size(int64_t head_dim) {
  ql_host::Device dev;
  if (ql_host::current(&dev) != QL_OK) return 0;
  switch (head_dim) {   // the largest of the variants' (equal for 8 and 4 bits)
    case 64: return std::max({stream_workspace<64, 8, 1>(dev.sms), stream_workspace<64, 8, 2>(dev.sms), tree_workspace<64, 8>(dev.sms)});
    case 128: return std::max({stream_workspace<128, 8, 1>(dev.sms), stream_workspace<128, 8, 2>(dev.sms), tree_workspace<128, 8>(dev.sms)});
    case 256: return std::max(stream_workspace<256, 8, 1>(dev.sms), stream_workspace<256, 8, 2>(dev.sms));
    default: return 0;
  }
}

}  // extern "C"
