// qshared.cu — C ABI of attention behind shared prefixes (declared in
// include/qlinear.h): one pass over the prefixes, each read once for all rows
// of its group, then one over what the requests have of their own, which takes
// the first one's sums and outputs in.  Both run the kernels of attention over
// the cache (qattend.cuh, qtree.cuh), each chosen for its own pass: a prefix
// has many rows a key, a request few.
#include "qattn_host.cuh"

extern "C" {

size_t ql_shared_attention_parts_size(int64_t total_q, int64_t q_heads, int64_t head_dim) {
  if (total_q < 0 || q_heads < 0 || head_dim < 0 || total_q > INT_MAX || q_heads > 65536 || head_dim > 256) return 0;
  // sums of the rows first, up to a multiple of 16 bytes
  const size_t rows = (size_t)total_q * (size_t)q_heads;
  return (rows * sizeof(float2) + 15) / 16 * 16 + rows * (size_t)head_dim * sizeof(float);
}

int ql_shared_attention(const ql_shared_attention_args* a, void* stream) {
  if (!a) return QL_ERR_NULL_POINTER;
  const bool some = a->own.batch > 0 && a->own.total_q > 0 && a->own.q_heads > 0;
  if (a->groups < 0 || a->groups > 65535 || a->prefix_width < 0 || a->prefix_width > INT_MAX) return QL_ERR_BAD_SHAPE;
  if (a->groups == 0) return ql_tree_attention(&a->own, stream);
  if (some) {
    if (!a->cu_group && a->groups != 1) return QL_ERR_BAD_SHAPE;
    if (!a->prefix_lens || !a->parts || (!a->prefix_table && a->prefix_width > 0)) return QL_ERR_NULL_POINTER;
    if (a->prefix_stride < a->prefix_width) return QL_ERR_BAD_STRIDE;
    if (!aligned(a->prefix_table, 4) || !aligned(a->prefix_lens, 4) || !aligned(a->cu_group, 4) || !aligned(a->parts, 16))
      return QL_ERR_UNSUPPORTED;
    if (a->parts_bytes < (int64_t)ql_shared_attention_parts_size(a->own.total_q, a->own.q_heads, a->own.cache.head_dim))
      return QL_ERR_WORKSPACE;
  }
  Attention own;
  bool nothing;
  int st = make_attention(&a->own, stream, &own, &nothing);
  if (st != QL_OK || nothing) return st;
  const int64_t rows = a->own.total_q * a->own.q_heads, head_dim = a->own.cache.head_dim;
  own.p.early_sums = static_cast<float2*>(a->parts);
  own.p.early_out = reinterpret_cast<float*>(static_cast<char*>(a->parts) + (rows * sizeof(float2) + 15) / 16 * 16);
  own.p.requests = (int)a->own.batch;
  Attention first = own;
  first.p.first_pass = 1;
  first.p.out = nullptr;
  first.p.lse = nullptr;
  first.p.mask = nullptr;
  first.p.mask_words = 0;
  first.p.page_table = static_cast<const int*>(a->prefix_table);
  first.p.kv_lens = static_cast<const int*>(a->prefix_lens);
  first.p.cu_group = static_cast<const int*>(a->cu_group);
  first.p.table_stride = a->prefix_stride;
  first.p.table_width = (int)a->prefix_width;
  first.p.batch = (int)a->groups;
  // one group may hold all rows; the choice of the kernel goes by their mean
  first.max_q = a->own.total_q;
  first.max_kv = std::min(std::max<int64_t>(a->max_prefix, 1), a->prefix_width * a->own.cache.page_size);
  first.max_rows = first.mean_rows = cdiv(a->own.total_q * own.p.group, a->groups);
  if ((st = run_attention<true>(first, head_dim, a->own.dtype)) != QL_OK) return st;
  return run_attention<true>(own, head_dim, a->own.dtype);
}

}  // extern "C"
