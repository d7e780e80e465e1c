// qattend.cuh — attention of a few new tokens per request (one, a chain, or a
// tree of drafted ones) over the quantised paged cache (sm_100a).
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(s_ij) / sum_j exp(s_ij),   s_ij = scale * q_i . k_j
// over the cached positions j that row i sees.  A request's last q_len cached
// positions are its new tokens; row i sees every position before them and,
// of them, those up to i (no mask) or those whose bit is set in its mask row.
// A row that sees nothing gives zeros and a log-sum of minus infinity.
#pragma once

#include "qcache.cuh"

namespace ql {
namespace att {

struct Params {
  kvc::Pool cache;
  kvc::Rows q;                   // [total_q][q_heads][head_dim]
  void* out;                     // same shape, contiguous
  float* lse;                    // [total_q][q_heads] or null
  const int* page_table;         // [batch][table_stride]
  const int* kv_lens;            // [batch]
  const int* cu_q;               // [batch + 1], or null: total_q / batch tokens each
  const unsigned long long* mask;  // [total_q][mask_words] or null
  long long table_stride;
  int table_width, num_pages;
  int batch, total_q, q_heads, group, mask_words;
  float scale;
  unsigned* err;
};

struct Request {
  int q0, q_len, kv_len;
};
__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  if (p.cu_q) {
    r.q0 = min(max(p.cu_q[b], 0), p.total_q);
    r.q_len = min(max(p.cu_q[b + 1], r.q0), p.total_q) - r.q0;
  } else {
    r.q_len = p.total_q / p.batch;
    r.q0 = b * r.q_len;
  }
  const long long most = min((long long)p.table_width << p.cache.page_shift, 0x7FFFFFFFll);
  r.kv_len = (int)min((long long)max(p.kv_lens[b], 0), most);
  return r;
}
__device__ __forceinline__ bool sees(const Params& p, const Request& r, int i, int j) {
  const int d = j - (r.kv_len - r.q_len);        // which new token position j is
  if (!p.mask) return d <= i;
  if (d < 0) return true;
  return d < 64 * p.mask_words && ((p.mask[(long long)(r.q0 + i) * p.mask_words + (d >> 6)] >> (d & 63)) & 1);
}

constexpr int kTile = 128;

// One CTA per (query head, new token): each thread scores one key of a tile of
// 128, then sums one element of the output over the tile.
template <typename T, int D>
__global__ void __launch_bounds__(kTile) simple_kernel(const Params p) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float q[D], w[kTile], red[4];
  const int head = blockIdx.x, token = blockIdx.y, t = threadIdx.x;
  const kvc::Pool& kv = p.cache;
  Request r;
  int b = 0;
  for (; b < p.batch; ++b) {
    r = request(p, b);
    if (token >= r.q0 && token < r.q0 + r.q_len) break;
  }
  if (b == p.batch) return;
  const int row = token - r.q0, kv_head = head / p.group;
  for (int d = t; d < D; d += kTile)
    q[d] = kvc::to_f(static_cast<const T*>(p.q.p)[(long long)token * p.q.token_stride + head * p.q.head_stride + d]);
  __syncthreads();
  const int span = kv.groups > 1 ? kvc::kGroup4 : D;
  constexpr int E = (D + kTile - 1) / kTile;
  float m = -INFINITY, l = 0.f, o[E] = {};
  for (int j0 = 0; j0 < r.kv_len; j0 += kTile) {
    const int j = j0 + t;
    float s = -INFINITY;
    if (j < r.kv_len && sees(p, r, row, j)) {
      const int page = p.page_table[b * p.table_stride + (j >> kv.page_shift)];
      if (page >= 0 && page < p.num_pages) {
        const kvc::RowAt k = kvc::row_at(kv, ((long long)page << kv.page_shift) + (j & ((1 << kv.page_shift) - 1)),
                                         kv_head, false);
        s = 0.f;
        for (int g = 0; g < kv.groups; ++g) {
          float sum = 0.f, f[8];
          for (int d = g * span; d < g * span + span; d += 8) {
            kvc::codes8(f, k.codes + d / 8 * kv.bits, kv.bits);
            #pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(f[i], q[d + i], sum);
          }
          s = fmaf(sum, kvc::bf16_bits_to_f(k.scales[g]), s);
        }
        s *= p.scale;
      } else {
        atomicCAS(p.err, 0u, (unsigned)kDevErrBadIndex);
      }
    }
    float top = s;
    #pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    if ((t & 31) == 0) red[t >> 5] = top;
    __syncthreads();
    const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    const float keep = m == -INFINITY ? 0.f : __expf(m - mn);
    w[t] = s == -INFINITY ? 0.f : expf(s - mn);
    __syncthreads();
    m = mn;
    l *= keep;
    for (int i = 0; i < kTile; ++i) l += w[i];
    #pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = e * kTile + t;
      o[e] *= keep;
      for (int i = 0; i < kTile && d < D; ++i) {
        if (w[i] == 0.f) continue;
        const int jj = j0 + i, page = p.page_table[b * p.table_stride + (jj >> kv.page_shift)];
        const kvc::RowAt v = kvc::row_at(kv, ((long long)page << kv.page_shift) + (jj & ((1 << kv.page_shift) - 1)),
                                         kv_head, true);
        const float c = kv.bits == 8 ? (float)(signed char)v.codes[d]
                                     : (float)((int)((v.codes[d >> 1] >> (4 * (d & 1))) & 15) - 8);
        o[e] = fmaf(w[i] * kvc::bf16_bits_to_f(v.scales[kv.groups > 1 ? d / kvc::kGroup4 : 0]), c, o[e]);
      }
    }
    __syncthreads();
  }
  #pragma unroll
  for (int e = 0; e < E; ++e)
    if (e * kTile + t < D)
      static_cast<T*>(p.out)[((long long)token * p.q_heads + head) * D + e * kTile + t] =
          kvc::from_f<T>(l == 0.f ? 0.f : o[e] / l);
  if (p.lse && t == 0) p.lse[(long long)token * p.q_heads + head] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace att
}  // namespace ql
