// qcache.cuh — rotary positions, and the quantised paged key/value cache:
// writing rows (with the rotation of q and k in the same launch) and reading
// them back (sm_100a).
//
// Rotary positions.  Pair i of a head at position p turns by the angle whose
// cosine and sine are table[p][i]:
//   y1 = x1 cos - x2 sin,   y2 = x2 cos + x1 sin,
// with (x1, x2) = (x[i], x[i + r/2]) in the half layout and (x[2i], x[2i+1])
// in the interleaved one; elements from r on pass through.  The inverse
// turns by the negative angle: the transpose, and so the gradient's direction,
// whatever factor the table has on its cosines and sines.  Computed in fp32 with every product and sum rounded
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

// Two neighbouring elements in a word.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ void unpack2(float& lo, float& hi, uint32_t v);
template <> __device__ __forceinline__ void unpack2<__half>(float& lo, float& hi, uint32_t v) {
  const float2 f = h2_to_f2(v);
  lo = f.x;
  hi = f.y;
}
template <> __device__ __forceinline__ void unpack2<__nv_bfloat16>(float& lo, float& hi, uint32_t v) {
  lo = __uint_as_float(v << 16);
  hi = __uint_as_float(v & 0xFFFF0000u);
}

template <typename T> struct alignas(8) Vec4 { T v[4]; };
template <typename T> struct alignas(16) Vec8 { T v[8]; };

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
// A chunk as it lies in memory: the run at oa (x, y), then the one at ob.
// `vec`: rows start on 16 bytes, so that runs are read and written at once.
template <typename T>
__device__ __forceinline__ uint4 load_chunk(const T* row, const Chunk& k, bool vec) {
  if (vec) {
    if (k.ob == k.oa + 4) return *reinterpret_cast<const uint4*>(row + k.oa);
    const uint2 a = *reinterpret_cast<const uint2*>(row + k.oa), b = *reinterpret_cast<const uint2*>(row + k.ob);
    return make_uint4(a.x, a.y, b.x, b.y);
  }
  const unsigned short *a = reinterpret_cast<const unsigned short*>(row + k.oa),
                       *b = reinterpret_cast<const unsigned short*>(row + k.ob);
  return make_uint4(a[0] | (unsigned)a[1] << 16, a[2] | (unsigned)a[3] << 16, b[0] | (unsigned)b[1] << 16,
                    b[2] | (unsigned)b[3] << 16);
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* row, const float (&a)[4], const float (&b)[4], const Chunk& k,
                                            bool vec) {
  const uint4 v = make_uint4(pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]), pack2<T>(b[0], b[1]), pack2<T>(b[2], b[3]));
  if (vec && k.ob == k.oa + 4) {
    *reinterpret_cast<uint4*>(row + k.oa) = v;
  } else if (vec) {
    *reinterpret_cast<uint2*>(row + k.oa) = make_uint2(v.x, v.y);
    *reinterpret_cast<uint2*>(row + k.ob) = make_uint2(v.z, v.w);
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      row[k.oa + i] = from_f<T>(a[i]);
      row[k.ob + i] = from_f<T>(b[i]);
    }
  }
}

// cos and sin of a chunk's four pairs: cos, sin, cos, sin of pairs 0 and 1, of 2 and 3.
struct Angles {
  float4 u, w;
};
// The inverse's sines are negative: exact, so that the products need not know.
__device__ __forceinline__ Angles load_angles(const float2* angles, int c, int inverse) {
  const float4* p = reinterpret_cast<const float4*>(angles + 4 * c);
  Angles t = {__ldg(p), __ldg(p + 1)};
  if (inverse) t = {{t.u.x, -t.u.y, t.u.z, -t.u.w}, {t.w.x, -t.w.y, t.w.z, -t.w.w}};
  return t;
}

__device__ __forceinline__ void turn_pair(float& x1, float& x2, float c, float s) {
  const float y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
  const float y2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
  x1 = y1;
  x2 = y2;
}
template <bool INTERLEAVED>
__device__ __forceinline__ void turn_chunk(float (&a)[4], float (&b)[4], const Angles& t) {
  if (INTERLEAVED) {
    turn_pair(a[0], a[1], t.u.x, t.u.y);
    turn_pair(a[2], a[3], t.u.z, t.u.w);
    turn_pair(b[0], b[1], t.w.x, t.w.y);
    turn_pair(b[2], b[3], t.w.z, t.w.w);
  } else {
    turn_pair(a[0], b[0], t.u.x, t.u.y);
    turn_pair(a[1], b[1], t.u.z, t.u.w);
    turn_pair(a[2], b[2], t.w.x, t.w.y);
    turn_pair(a[3], b[3], t.w.z, t.w.w);
  }
}
__device__ __forceinline__ void turn_chunk(float (&a)[4], float (&b)[4], const Angles& t, const Chunk& k,
                                           const Turn& turn) {
  if (!k.turns) return;
  if (turn.interleaved)
    turn_chunk<true>(a, b, t);
  else
    turn_chunk<false>(a, b, t);
}
template <typename T>
__device__ __forceinline__ void widen(float (&a)[4], float (&b)[4], const uint4& r) {
  unpack2<T>(a[0], a[1], r.x);
  unpack2<T>(a[2], a[3], r.y);
  unpack2<T>(b[0], b[1], r.z);
  unpack2<T>(b[2], b[3], r.w);
}

// The row of the table of position p; one outside it is recorded in the
// device error word and takes the nearest row.
__device__ __forceinline__ const float2* angles_of(const Turn& t, long long p, unsigned* err) {
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

// Division of numbers below 2^31 by one known on the host: with s the
// smallest power of two at least d and m = ceil(2^31 s / d), n m / (2^31 s)
// exceeds n / d by less than 1 / d, so its whole part is n / d's.
struct Divisor {
  unsigned m, shift;
  __device__ __forceinline__ int of(int n) const { return (int)(((unsigned long long)(unsigned)n * m) >> shift); }
};

// -------------------------------------------------------------------- rotary
// How threads lie over (token, head, chunk): `beside` heads of a token side by
// side, `tokens` tokens to a CTA.
struct Grid {
  int beside, tokens, chunks;      // chunks = head_dim / 8
  Divisor by_token, by_chunks;     // by beside * chunks, by chunks
};
struct Place {
  int token, head, c;              // token -1: none
};
__device__ __forceinline__ Place place_of(const Grid& g, int cta, int total) {
  const int mine = g.by_token.of(threadIdx.x), rest = threadIdx.x - mine * g.beside * g.chunks;
  const int token = cta * g.tokens + mine, head = g.by_chunks.of(rest);
  return {mine < g.tokens && token < total ? token : -1, head, rest - head * g.chunks};
}

// Bound by memory, and by the chain behind a token: its position, then its
// angles.  A thread keeps one chunk of 8 elements, and so its angles, over
// kHeads heads whose loads are all in flight before the angles are waited for.
constexpr int kHeads = 4;
struct RotaryParams {
  Turn turn;
  Rows x, out;
  Grid grid;
  int tokens, heads;
  unsigned* err;
};
// WHOLE_HALF: half layout, whole heads, 16-byte aligned rows; the questions
// that each head of the general body asks are then settled.  By this body and
// by the general one, 16384 tokens of 32 heads of 128: 45.7 us, 49.3; of 64
// heads of 64: 47.8, 48.9; 4096 of 40 heads of 256: 35.3, 34.4; an append of
// 8192 x (32 + 8 + 8) x 128: 44.1, 46.5.  For what else there is, bodies of
// their own lost: interleaved 50.9 against 49.8, a part of the heads (where a
// warp's chunks differ) 5.5 against 4.5.
template <typename T, bool WHOLE_HALF>
__device__ __forceinline__ void rotate_rows(const RotaryParams& p, const Place& at) {
  const Chunk k = WHOLE_HALF ? Chunk{4 * at.c, 4 * (p.grid.chunks + at.c), true} : chunk_of(at.c, p.turn, true);
  const long long x_step = p.grid.beside * p.x.head_stride, out_step = p.grid.beside * p.out.head_stride;
  const T* x = static_cast<const T*>(p.x.p) + at.token * p.x.token_stride + at.head * p.x.head_stride;
  T* out = static_cast<T*>(const_cast<void*>(p.out.p)) + at.token * p.out.token_stride + at.head * p.out.head_stride;
  const long long position = k.turns ? load_index(p.turn.positions, at.token, p.turn.wide) : 0;
  Angles angles = {};
  auto load = [&](const T* row) {
    if (!WHOLE_HALF) return load_chunk(row, k, p.x.vec);
    const uint2 a = *reinterpret_cast<const uint2*>(row + k.oa), b = *reinterpret_cast<const uint2*>(row + k.ob);
    return make_uint4(a.x, a.y, b.x, b.y);
  };
  auto turn_and_store = [&](T* row, const uint4& raw) {
    float a[4], b[4];
    widen<T>(a, b, raw);
    if (WHOLE_HALF)
      turn_chunk<false>(a, b, angles);
    else
      turn_chunk(a, b, angles, k, p.turn);
    if (WHOLE_HALF) {
      *reinterpret_cast<uint2*>(row + k.oa) = make_uint2(pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]));
      *reinterpret_cast<uint2*>(row + k.ob) = make_uint2(pack2<T>(b[0], b[1]), pack2<T>(b[2], b[3]));
    } else {
      store_chunk(row, a, b, k, p.out.vec);
    }
  };
  for (int h = at.head; h < p.heads; h += kHeads * p.grid.beside) {
    const bool all = WHOLE_HALF && h + (kHeads - 1) * p.grid.beside < p.heads;
    uint4 raw[kHeads];
    if (all) {
      #pragma unroll
      for (int i = 0; i < kHeads; ++i) raw[i] = load(x + i * x_step);
    } else {
      #pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (h + i * p.grid.beside < p.heads) raw[i] = load(x + i * x_step);
    }
    if (h == at.head && k.turns) angles = load_angles(angles_of(p.turn, position, p.err), at.c, p.turn.inverse);
    if (all) {
      #pragma unroll
      for (int i = 0; i < kHeads; ++i) turn_and_store(out + i * out_step, raw[i]);
    } else {
      #pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (h + i * p.grid.beside < p.heads) turn_and_store(out + i * out_step, raw[i]);
    }
    x += kHeads * x_step;
    out += kHeads * out_step;
  }
}
template <typename T>
__device__ __forceinline__ void rotate_heads(const RotaryParams& p, int cta) {
  const Place at = place_of(p.grid, cta, p.tokens);
  if (at.token < 0) return;
  if (p.x.vec && p.out.vec && !p.turn.interleaved && p.turn.rotary_dim == 8 * p.grid.chunks)
    rotate_rows<T, true>(p, at);
  else
    rotate_rows<T, false>(p, at);
}
// Bound by reading and writing the heads once.  16384 tokens of 32 heads of
// 128 (277 MB with the angles): 46 us in the half layout, 48 interleaved, 6.1
// and 5.8 TB/s, where a plain copy reaches 6.5; one token: 1.8 us, a launch.
template <typename T>
__global__ void __launch_bounds__(256, 5) rotary_kernel(const RotaryParams p) {
  griddep_launch_dependents();
  griddep_wait();
  rotate_heads<T>(p, blockIdx.x);
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
  RotaryParams q;          // the queries, whose turn is the keys' too (rotary_dim 0: no key turns, and there are no queries)
  Pool cache;
  Rows k, v;
  Grid grid;               // of the keys and values
  const void* slots;
  int wide_slots, tokens;
  int kv_ctas;             // the CTAs before those of the queries
};

// Codes of four elements against a scale that is positive and finite, and
// inv = 1 / s: rne(x / s) without a division.  x inv is within 2^-22 of x / s
// relatively, 2^-15 where codes can differ (below 128), so it rounds alike
// unless it is that close to half way between two codes; those few elements
// are divided.  A row whose scale is below 2^-125 comes with inv = infinity and
// is divided whole: there bf16 can round the scale far down, and only the clamp
// keeps its codes in range.  A larger scale is a normal number, rounded to 8
// bits: at least max|x| / top * (1 - 2^-8), so x / s is below top + 1/2 and
// needs no clamp.  Adding 1.5 * 2^23 leaves the rounded integer in the low bits.
template <int BITS>
__device__ __forceinline__ unsigned quantise4(const float (&f)[4], float s, float inv) {
  constexpr float kRound = 12582912.f;
  constexpr float top = BITS == 8 ? 127.f : 7.f;
  unsigned q[4];
  bool close = !(inv < INFINITY);
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = __fmul_rn(f[i], inv);
    const float r = __fadd_rn(y, kRound);
    q[i] = __float_as_uint(r);
    close |= fabsf(__fsub_rn(y, __fsub_rn(r, kRound))) > 0.5f - 0x1p-14f;
  }
  if (close) {
    #pragma unroll
    for (int i = 0; i < 4; ++i)
      q[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fdiv_rn(f[i], s), -top), top), kRound));
  }
  if constexpr (BITS == 8) {
    return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = (q[i] + 8u) & 15u;
    return q[0] | q[1] << 4 | q[2] << 8 | q[3] << 12;
  }
}

// One row to its slot: LANES neighbouring lanes hold it and reduce its maxima
// by shuffles, which all lanes of the warp take part in; `live` lanes write.
template <int LANES, int BITS>
__device__ __forceinline__ void store_row(const RowAt& dst, const float (&a)[4], const float (&b)[4], const Chunk& k,
                                          int c, bool live) {
  constexpr int kGroups = BITS == 8 ? 1 : LANES * 8 / kGroup4;
  // |x| as ordered integers: an infinity or NaN ends up as the maximum
  unsigned ma = 0, mb = 0;
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    ma = max(ma, __float_as_uint(a[i]) & 0x7FFFFFFFu);
    mb = max(mb, __float_as_uint(b[i]) & 0x7FFFFFFFu);
  }
  const int ga = kGroups > 1 ? k.oa / kGroup4 : 0, gb = kGroups > 1 ? k.ob / kGroup4 : 0;
  float sa = 0.f, sb = 0.f;
  #pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    unsigned m = kGroups == 1 ? max(ma, mb) : max(ga == g ? ma : 0u, gb == g ? mb : 0u);
    #pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    constexpr float kInvTop = BITS == 8 ? (float)(1.0 / 127.0) : (float)(1.0 / 7.0);
    const unsigned short s16 = __bfloat16_as_ushort(__float2bfloat16_rn(__fmul_rn(__uint_as_float(m), kInvTop)));
    const float s = bf16_bits_to_f(s16);
    if (ga == g) sa = s;
    if (gb == g) sb = s;
    if (live && c == 0) dst.scales[g] = s16;
  }
  if (!live) return;
  // a scale below 2^-125 has no reciprocal in fp32's normal range: such rows are divided
  constexpr unsigned kNone = BITS == 8 ? 0u : 0x8888u;
  const bool fa = sa > 0.f && sa < INFINITY, fb = sb > 0.f && sb < INFINITY;
  const float ia = sa >= 0x1p-125f ? __frcp_rn(sa) : INFINITY;
  const float ib = kGroups == 1 || sb == sa ? ia : sb >= 0x1p-125f ? __frcp_rn(sb) : INFINITY;
  const unsigned qa = fa ? quantise4<BITS>(a, sa, ia) : kNone, qb = fb ? quantise4<BITS>(b, sb, ib) : kNone;
  if (BITS == 8) {
    if (k.ob == k.oa + 4) {
      *reinterpret_cast<uint2*>(dst.codes + k.oa) = make_uint2(qa, qb);
    } else {
      *reinterpret_cast<unsigned*>(dst.codes + k.oa) = qa;
      *reinterpret_cast<unsigned*>(dst.codes + k.ob) = qb;
    }
  } else if (k.ob == k.oa + 4) {
    *reinterpret_cast<unsigned*>(dst.codes + k.oa / 2) = qa | qb << 16;
  } else {
    *reinterpret_cast<unsigned short*>(dst.codes + k.oa / 2) = (unsigned short)qa;
    *reinterpret_cast<unsigned short*>(dst.codes + k.ob / 2) = (unsigned short)qb;
  }
}

// The first CTAs write keys and values, LANES = head_dim / 8 lanes taking the
// key and the value row of a head; the others turn the queries.  Spread among
// the queries' CTAs instead, those of keys and values gain 1 % at 8192 tokens
// and lose 3 % at 2501.  Queries are bound by memory; keys and values by the
// instructions that a code takes.  8192 tokens, 32 + 8 + 8 heads of 128, fp16:
// 44 us at 8 bits (4.3 TB/s) and 47 at 4; without queries 21.5 us (2.6 TB/s).
template <typename T, int LANES, int BITS>
__global__ void __launch_bounds__(256, 4) append_kernel(const AppendParams p) {
  griddep_launch_dependents();
  griddep_wait();
  if ((int)blockIdx.x >= p.kv_ctas) {
    rotate_heads<T>(p.q, blockIdx.x - p.kv_ctas);
    return;
  }
  const Pool& kv = p.cache;
  const Turn& turn = p.q.turn;
  const Place at = place_of(p.grid, blockIdx.x, p.tokens);
  const int token = max(at.token, 0);
  const Chunk straight = chunk_of(at.c, turn, false), turned = chunk_of(at.c, turn, turn.rotary_dim > 0);
  long long slot = load_index(p.slots, token, p.wide_slots);
  const long long position = turned.turns ? load_index(turn.positions, token, turn.wide) : 0;
  Angles angles = {};
  for (int first = 0; first < kv.heads; first += p.grid.beside) {       // every lane: the shuffles want them all
    const int h = min(first + at.head, kv.heads - 1);
    const uint4 k_raw = load_chunk(static_cast<const T*>(p.k.p) + token * p.k.token_stride + h * p.k.head_stride, turned, p.k.vec);
    const uint4 v_raw = load_chunk(static_cast<const T*>(p.v.p) + token * p.v.token_stride + h * p.v.head_stride, straight, p.v.vec);
    if (first == 0) {
      if (turned.turns) angles = load_angles(angles_of(turn, position, p.q.err), at.c, turn.inverse);
      if (at.token < 0) slot = -1;
      if (slot >= kv.slots) {
        atomicCAS(p.q.err, 0u, (unsigned)kDevErrBadIndex);
        slot = -1;
      }
    }
    const bool live = slot >= 0 && first + at.head < kv.heads;
    const long long where = max(slot, 0ll);
    float a[4], b[4];
    widen<T>(a, b, k_raw);
    turn_chunk(a, b, angles, turned, turn);
    store_row<LANES, BITS>(row_at(kv, where, h, false), a, b, turned, at.c, live);
    widen<T>(a, b, v_raw);
    store_row<LANES, BITS>(row_at(kv, where, h, true), a, b, straight, at.c, live);
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
__device__ __forceinline__ void codes8(float (&f)[8], uint2 w, int bits) {
  if (bits == 8) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = (float)(int)(signed char)(w.x >> (8 * i));
      f[4 + i] = (float)(int)(signed char)(w.y >> (8 * i));
    }
  } else {
    #pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)((int)((w.x >> (4 * i)) & 15u) - 8);
  }
}

// A thread takes 8 elements of the key and of the value row of kTokens tokens,
// 256 / (heads * chunks) apart or more, so that 2 kTokens loads are in flight:
// CTA i has tokens i * span .., span = tokens side by side * kTokens.  Bound by
// memory, most of it what is written: 128032 rows of 8 heads of 128 at 4 bits
// take 89 us, 5.2 TB/s.
constexpr int kTokens = 4;
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const ReadParams p, int log_chunks, int side, int split) {
  griddep_launch_dependents();
  griddep_wait();
  const Pool& kv = p.cache;
  // part of a token's heads * chunks that this CTA has (all of it where split is 1), and the token of the thread
  const int per_token = kv.heads << log_chunks;
  const int part = split > 1 ? blockIdx.x % split : 0;
  const long long group = split > 1 ? blockIdx.x / split : blockIdx.x;
  const int beside = split > 1 ? 0 : threadIdx.x / per_token;
  const int at = split > 1 ? part * 256 + threadIdx.x : threadIdx.x - beside * per_token;
  if (beside >= side || at >= per_token) return;
  const int head = at >> log_chunks, c = at & ((1 << log_chunks) - 1);
  const long long first = group * side * kTokens + beside;
  long long slot[kTokens];
  #pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    const long long token = first + i * side;
    slot[i] = token < p.tokens ? load_index(p.slots, token, p.wide_slots) : -1;
    if (slot[i] >= kv.slots) {
      atomicCAS(p.err, 0u, (unsigned)kDevErrBadIndex);
      slot[i] = -1;
    }
  }
  uint2 w[kTokens][2];
  unsigned short s[kTokens][2];
  #pragma unroll
  for (int i = 0; i < kTokens; ++i)
    #pragma unroll
    for (int v = 0; v < 2; ++v) {
      w[i][v] = make_uint2(0u, 0u);
      s[i][v] = 0;
      if (slot[i] >= 0) {
        const RowAt r = row_at(kv, slot[i], head, v != 0);
        if (kv.bits == 8)
          w[i][v] = *reinterpret_cast<const uint2*>(r.codes + c * 8);
        else
          w[i][v].x = *reinterpret_cast<const unsigned*>(r.codes + c * 4);
        s[i][v] = r.scales[kv.groups > 1 ? c * 8 / kGroup4 : 0];
      }
    }
  #pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    const long long token = first + i * side;
    if (token >= p.tokens) break;
    #pragma unroll
    for (int v = 0; v < 2; ++v) {
      float f[8];
      codes8(f, w[i][v], kv.bits);
      const float scale = bf16_bits_to_f(s[i][v]);
      *reinterpret_cast<uint4*>(static_cast<T*>(v ? p.v : p.k) + ((token * per_token + at) << 3)) =
          make_uint4(pack2<T>(f[0] * scale, f[1] * scale), pack2<T>(f[2] * scale, f[3] * scale),
                     pack2<T>(f[4] * scale, f[5] * scale), pack2<T>(f[6] * scale, f[7] * scale));
    }
  }
}

}  // namespace kvc
}  // namespace ql
