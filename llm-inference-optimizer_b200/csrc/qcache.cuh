// qcache.cuh — rotary positions, and the quantised paged key/value cache:
// writing rows (with the rotation of q and k in the same launch) and reading
// them back (sm_100a).
//
// Rotary positions.  Pair i of a head at position p turns by the angle whose
// cosine and sine are table[p][i]:
//   y1 = x1 cos - x2 sin,   y2 = x2 cos + x1 sin,
// with (x1, x2) = (x[i], x[i + r/2]) in the half layout and (x[2i], x[2i+1])
// in the interleaved one; elements from r on pass through.  The inverse
// turns by the negative angle; the rotation being orthogonal, it is also the
// gradient's direction.  Computed in fp32 with every product and sum rounded
// on its own (no contraction), so that a row quantised from it has the codes
// that the same expression gives elementwise elsewhere.
//
// A cached row is one token of one key/value head: integer codes and a bf16
// scale per group (the whole row at 8 bits, 64 elements at 4 bits):
//   s = bf16(max|x| * (1 / top)),  q = clamp(rne(x / s), -top, top),
// top = 127 or 7.  bf16 keeps fp32's range, so no finite input overflows the
// scale or needs a floor; its 8 significant bits cost nothing, because the
// codes are taken against the rounded scale.  A group whose scale is zero or
// not finite has codes of zero: it reads back as zeros, or as NaN when an
// input was infinite or NaN.  4-bit codes are stored as q + 8, the even
// element in the low nibble.
//
// Layout: codes [page][head][page_size][row bytes], scales [page][head]
// [page_size][groups]; a slot is page * page_size + offset.
#pragma once

#include <cuda_bf16.h>

#include "ql_common.cuh"

namespace ql {
namespace kvc {

constexpr int kGroup4 = 64;          // elements that share a scale at 4 bits

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
__device__ __forceinline__ float bf16_bits_to_f(unsigned short b) { return __uint_as_float((unsigned)b << 16); }

template <typename T> struct alignas(8) Vec4 { T v[4]; };
template <typename T> struct alignas(16) Vec8 { T v[8]; };

// Four neighbouring elements, in one access where `vec` says that rows are
// 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load4(float (&f)[4], const T* p, bool vec) {
  if (vec) {
    const Vec4<T> a = *reinterpret_cast<const Vec4<T>*>(p);
    #pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_f(a.v[i]);
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_f(p[i]);
  }
}
template <typename T>
__device__ __forceinline__ void load8(float (&a)[4], float (&b)[4], const T* p, bool vec) {
  if (vec) {
    const Vec8<T> x = *reinterpret_cast<const Vec8<T>*>(p);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = to_f(x.v[i]);
      b[i] = to_f(x.v[4 + i]);
    }
  } else {
    load4(a, p, false);
    load4(b, p + 4, false);
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&f)[4], bool vec) {
  Vec4<T> a;
  #pragma unroll
  for (int i = 0; i < 4; ++i) a.v[i] = from_f<T>(f[i]);
  if (vec) {
    *reinterpret_cast<Vec4<T>*>(p) = a;
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = a.v[i];
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&a)[4], const float (&b)[4], bool vec) {
  if (vec) {
    Vec8<T> x;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      x.v[i] = from_f<T>(a[i]);
      x.v[4 + i] = from_f<T>(b[i]);
    }
    *reinterpret_cast<Vec8<T>*>(p) = x;
  } else {
    store4(p, a, false);
    store4(p + 4, b, false);
  }
}

__device__ __forceinline__ long long load_index(const void* p, long long i, int wide) {
  return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

struct Turn {
  const float2* table;     // [max_positions][rotary_dim / 2] (cos, sin)
  const void* positions;   // [tokens], 4 or 8 bytes each
  long long max_positions;
  int wide;                // positions are 8 bytes
  int rotary_dim;          // a multiple of 8; 0: nothing turns
  int interleaved;
  int inverse;
};

// Which 8 elements of a head chunk c covers: two runs of 4 at oa and ob.
// Chunks below rotary_dim / 8 hold four pairs.
struct Chunk {
  int oa, ob;
  bool turns;
};
__device__ __forceinline__ Chunk chunk_of(int c, const Turn& t, bool rotate) {
  Chunk k;
  k.turns = rotate && c < (t.rotary_dim >> 3);
  const bool split = k.turns && !t.interleaved;
  k.oa = split ? 4 * c : 8 * c;
  k.ob = split ? (t.rotary_dim >> 1) + 4 * c : 8 * c + 4;
  return k;
}
template <typename T>
__device__ __forceinline__ void load_chunk(float (&a)[4], float (&b)[4], const T* row, const Chunk& k, bool vec) {
  if (k.ob == k.oa + 4) {
    load8(a, b, row + k.oa, vec);
  } else {
    load4(a, row + k.oa, vec);
    load4(b, row + k.ob, vec);
  }
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* row, const float (&a)[4], const float (&b)[4], const Chunk& k,
                                            bool vec) {
  if (k.ob == k.oa + 4) {
    store8(row + k.oa, a, b, vec);
  } else {
    store4(row + k.oa, a, vec);
    store4(row + k.ob, b, vec);
  }
}

// cos and sin of the chunk's four pairs.
__device__ __forceinline__ void load_angles(float (&cs)[4], float (&sn)[4], const float2* angles, int c,
                                            int inverse) {
  const float4* p = reinterpret_cast<const float4*>(angles + 4 * c);
  const float4 u = __ldg(p), w = __ldg(p + 1);
  const float m = inverse ? -1.f : 1.f;
  cs[0] = u.x; sn[0] = m * u.y; cs[1] = u.z; sn[1] = m * u.w;
  cs[2] = w.x; sn[2] = m * w.y; cs[3] = w.z; sn[3] = m * w.w;
}

__device__ __forceinline__ void turn_pair(float& x1, float& x2, float c, float s) {
  const float y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
  const float y2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
  x1 = y1;
  x2 = y2;
}
__device__ __forceinline__ void turn_chunk(float (&a)[4], float (&b)[4], const float (&cs)[4],
                                           const float (&sn)[4], int interleaved) {
  if (interleaved) {
    turn_pair(a[0], a[1], cs[0], sn[0]);
    turn_pair(a[2], a[3], cs[1], sn[1]);
    turn_pair(b[0], b[1], cs[2], sn[2]);
    turn_pair(b[2], b[3], cs[3], sn[3]);
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) turn_pair(a[i], b[i], cs[i], sn[i]);
  }
}

// The token's row of the table; a position outside it is recorded in the
// device error word and takes the nearest row.
__device__ __forceinline__ const float2* angles_of(const Turn& t, long long token, unsigned* err) {
  long long p = load_index(t.positions, token, t.wide);
  if (p < 0 || p >= t.max_positions) {
    atomicCAS(err, 0u, (unsigned)kDevErrBadIndex);
    p = p < 0 ? 0 : t.max_positions - 1;
  }
  return t.table + p * (t.rotary_dim >> 1);
}

struct Rows {              // [tokens][heads][head_dim] with strides in elements
  const void* p;
  long long token_stride, head_stride;
  int vec;                 // every row starts on 16 bytes
};

// -------------------------------------------------------------------- rotary
struct RotaryParams {
  Turn turn;
  Rows x, out;
  long long tokens;
  int heads, chunks;       // chunks = head_dim / 8
  unsigned* err;
};

// One CTA per token; a thread takes chunks of 8 elements across the heads.
template <typename T>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const long long token = blockIdx.x;
  const float2* angles = angles_of(p.turn, token, p.err);
  const int n = p.heads * p.chunks;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int h = i / p.chunks, c = i - h * p.chunks;
    const Chunk k = chunk_of(c, p.turn, true);
    float a[4], b[4], cs[4], sn[4];
    load_chunk(a, b, static_cast<const T*>(p.x.p) + token * p.x.token_stride + h * p.x.head_stride, k, p.x.vec);
    if (k.turns) {
      load_angles(cs, sn, angles, c, p.turn.inverse);
      turn_chunk(a, b, cs, sn, p.turn.interleaved);
    }
    T* row = static_cast<T*>(const_cast<void*>(p.out.p)) + token * p.out.token_stride + h * p.out.head_stride;
    store_chunk(row, a, b, k, p.out.vec);
  }
}

// --------------------------------------------------------------------- cache
struct Pool {              // strides between pages in bytes (codes) and elements (scales), below 2^32
  unsigned char *k_codes, *v_codes;
  unsigned short *k_scales, *v_scales;
  unsigned k_page, v_page, ks_page, vs_page;
  long long slots;         // pages * page_size
  int page_shift;          // log2(page_size)
  int heads, row_bytes, groups, bits;
};
struct RowAt {
  unsigned char* codes;
  unsigned short* scales;
};
__device__ __forceinline__ RowAt row_at(const Pool& c, long long slot, int head, bool value) {
  const long long page = slot >> c.page_shift;
  const int at = (head << c.page_shift) + (int)(slot & ((1 << c.page_shift) - 1));
  RowAt r;
  r.codes = (value ? c.v_codes + page * c.v_page : c.k_codes + page * c.k_page) + (long long)at * c.row_bytes;
  r.scales = (value ? c.v_scales + page * c.vs_page : c.k_scales + page * c.ks_page) + (long long)at * c.groups;
  return r;
}

struct AppendParams {
  Turn turn;
  Pool cache;
  Rows q, q_out, k, v;
  const void* slots;
  int wide_slots;
  long long tokens;
  int q_heads;             // 0: no queries
  unsigned* err;
};

// Codes of four elements against a scale that is positive and finite.
__device__ __forceinline__ unsigned quantise4(const float (&f)[4], float s, int bits) {
  unsigned w = 0;
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float top = bits == 8 ? 127.f : 7.f;
    const int q = (int)fminf(fmaxf(rintf(__fdiv_rn(f[i], s)), -top), top);
    w |= bits == 8 ? (unsigned)(q & 0xFF) << (8 * i) : (unsigned)(q + 8) << (4 * i);
  }
  return w;
}

// One CTA per token; LANES = head_dim / 8 neighbouring lanes hold one row
// (query, key or value head) and reduce its maxima by shuffles.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const long long token = blockIdx.x;
  const Pool& kv = p.cache;
  const int lane = threadIdx.x % LANES, rows_per_pass = blockDim.x / LANES;
  const int total = p.q_heads + 2 * kv.heads;
  long long slot = load_index(p.slots, token, p.wide_slots);
  if (slot >= kv.slots) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0u, (unsigned)kDevErrBadIndex);
    slot = -1;
  }
  const bool rotary = p.turn.rotary_dim > 0;
  float cs[4], sn[4];
  if (rotary && lane < (p.turn.rotary_dim >> 3))
    load_angles(cs, sn, angles_of(p.turn, token, p.err), lane, p.turn.inverse);

  // every lane takes every pass, so that the shuffles find all lanes
  for (int first = 0; first < total; first += rows_per_pass) {
    const int row = first + threadIdx.x / LANES;
    const bool query = row < p.q_heads, value = row >= p.q_heads + kv.heads;
    const bool live = row < total && (query || slot >= 0);
    const int head = query ? row : row - p.q_heads - (value ? kv.heads : 0);
    const Chunk k = chunk_of(lane, p.turn, rotary && !value);
    float a[4] = {}, b[4] = {};
    if (live) {
      const Rows& src = query ? p.q : value ? p.v : p.k;
      load_chunk(a, b, static_cast<const T*>(src.p) + token * src.token_stride + head * src.head_stride, k,
                 src.vec);
      if (k.turns) turn_chunk(a, b, cs, sn, p.turn.interleaved);
    }
    if (live && query) {
      T* out = static_cast<T*>(const_cast<void*>(p.q_out.p)) + token * p.q_out.token_stride +
               head * p.q_out.head_stride;
      store_chunk(out, a, b, k, p.q_out.vec);
    }
    // |x| as ordered integers: an infinity or NaN ends up as the maximum
    unsigned ma = 0, mb = 0;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      ma = max(ma, __float_as_uint(a[i]) & 0x7FFFFFFFu);
      mb = max(mb, __float_as_uint(b[i]) & 0x7FFFFFFFu);
    }
    const int ga = kv.groups > 1 ? k.oa / kGroup4 : 0, gb = kv.groups > 1 ? k.ob / kGroup4 : 0;
    float sa = 0.f, sb = 0.f;
    #pragma unroll 1
    for (int g = 0; g < kv.groups; ++g) {
      unsigned m = max(ga == g ? ma : 0u, gb == g ? mb : 0u);
      #pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float inv_top = kv.bits == 8 ? (float)(1.0 / 127.0) : (float)(1.0 / 7.0);
      const unsigned short s16 = __bfloat16_as_ushort(__float2bfloat16_rn(__fmul_rn(__uint_as_float(m), inv_top)));
      const float s = bf16_bits_to_f(s16);
      if (ga == g) sa = s;
      if (gb == g) sb = s;
      if (live && !query && lane == 0) row_at(kv, slot, head, value).scales[g] = s16;
    }
    if (live && !query) {
      const bool fa = sa > 0.f && sa < INFINITY, fb = sb > 0.f && sb < INFINITY;
      const unsigned none = kv.bits == 8 ? 0u : 0x8888u;
      const unsigned qa = fa ? quantise4(a, sa, kv.bits) : none, qb = fb ? quantise4(b, sb, kv.bits) : none;
      unsigned char* codes = row_at(kv, slot, head, value).codes;
      if (kv.bits == 8) {
        *reinterpret_cast<unsigned*>(codes + k.oa) = qa;
        *reinterpret_cast<unsigned*>(codes + k.ob) = qb;
      } else {
        *reinterpret_cast<unsigned short*>(codes + k.oa / 2) = (unsigned short)qa;
        *reinterpret_cast<unsigned short*>(codes + k.ob / 2) = (unsigned short)qb;
      }
    }
  }
}

// ---------------------------------------------------------------------- read
struct ReadParams {
  Pool cache;
  const void* slots;
  int wide_slots;
  long long tokens;
  void *k, *v;             // [tokens][heads][head_dim], contiguous, 16-byte aligned
  unsigned* err;
};

// Codes of 8 elements as integers in fp32.
__device__ __forceinline__ void codes8(float (&f)[8], const unsigned char* p, int bits) {
  if (bits == 8) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = (float)(int)(signed char)(w.x >> (8 * i));
      f[4 + i] = (float)(int)(signed char)(w.y >> (8 * i));
    }
  } else {
    const unsigned w = *reinterpret_cast<const unsigned*>(p);
    #pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)((int)((w >> (4 * i)) & 15u) - 8);
  }
}

// A thread per 8 elements of a (token, head, key or value) row.
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const ReadParams p, int chunks) {
  griddep_launch_dependents();
  griddep_wait();
  const Pool& kv = p.cache;
  const long long n = p.tokens * kv.heads * chunks;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int c = (int)(i % chunks);
  const long long row = i / chunks;
  const long long token = row / kv.heads;
  const int head = (int)(row - token * kv.heads);
  const bool value = blockIdx.y != 0;
  const long long slot = load_index(p.slots, token, p.wide_slots);
  float f[8] = {};
  if (slot >= kv.slots) {
    atomicCAS(p.err, 0u, (unsigned)kDevErrBadIndex);
  } else if (slot >= 0) {
    const RowAt r = row_at(kv, slot, head, value);
    codes8(f, r.codes + c * kv.bits, kv.bits);
    const float s = bf16_bits_to_f(r.scales[kv.groups > 1 ? c * 8 / kGroup4 : 0]);
    #pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= s;
  }
  Vec8<T> o;
  #pragma unroll
  for (int j = 0; j < 8; ++j) o.v[j] = from_f<T>(f[j]);
  *reinterpret_cast<Vec8<T>*>(static_cast<T*>(value ? p.v : p.k) + i * 8) = o;
}

}  // namespace kvc
}  // namespace ql
