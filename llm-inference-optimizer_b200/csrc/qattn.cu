// qattn.cu — C ABI of the attention side of libqlinear.so (declared in
// include/qlinear.h): rotary positions, the quantised paged cache and
// attention over it.  Argument checks, variant choice and launches; every
// entry point returns a status and allocates nothing.
#include "qattn_host.cuh"

namespace {

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
  Attention work;
  bool nothing;
  const int st = make_attention(a, stream, &work, &nothing);
  return st != QL_OK || nothing ? st : run_attention<false>(work, a->cache.head_dim, a->dtype);
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
