// qsample.cuh — drawing a token from each row of logits, with temperature,
// top-k, top-p and min-p, by given random numbers (sm_100a).
//
// Token i of a row has weight w_i = exp((x_i - max) / T).  Tokens are ordered
// by their logit, equal ones by their index; of that order are kept
//   top-k  the first k,
//   top-p  those before which the kept weights come to less than p of their sum,
//   min-p  those with w_i >= m (m of the largest weight, which is 1),
// the first always.  The token drawn is the first, by index, at which the kept
// weights' running sum exceeds u times their sum W.  Its log-probability is
// log(w_i / W).  T <= 0 takes the first of the order.
//
// A cluster of CTAs shares a row.  Its first pass finds the largest logit; what
// comes next depends on the row's filters:
//   none            one pass sums the weights by blocks; the block that holds the
//                   token is then read again.
//   few are kept    a bound below the last token kept is found without reading the
//                   row again: each thread's largest logit stands for the others
//                   (k threads whose largest is >= v: k tokens are; if these tokens'
//                   weights come to p of the sum, the kept ones lie at v and above),
//                   and for min-p it is known.  One pass collects the tokens above
//                   it in one CTA, which sorts them and does the rest.
//   many are kept   all filters keep a beginning of the order, so what is kept is
//                   known by its last token: a value v and how many of the tokens
//                   equal to v are kept.  v is the largest value whose measure F(v)
//                   over tokens x >= v (their number; the sum of their weights)
//                   reaches a target.  For weights a histogram narrows it down to
//                   the tokens that one CTA sorts; else it is searched for over the
//                   type's values in their order, which are whole numbers, with
//                   four thresholds a round, each round a pass.
//
// A token is drawn, or not, by the comparison of two running sums, so these are
// held to more than fp32.  Sums over many weights are first taken, in fp64, of
// weights in fp32, which says how they compare unless they come closer than
// 2^-19.6 of themselves; then the weights are taken again in fp64.  The
// log-probability is of the sum that decided, off by up to 6e-7 (kOff).
//
// What bounds it: for few rows the chain of passes and meetings of the cluster (a
// meeting 0.5 us, each function's first run its way from memory: less code is
// quicker than unrolled code).  For many it is waiting too: a row's passes follow
// one another, first the largest logit and then the weights, a meeting behind each,
// and 256 rows of two CTAs are 1.73 rounds of the SMs' places; the instructions (a
// dozen a logit) take half of the issue slots.  Of spread-out logits 7 rows in 100
// want fp64, some 40 instructions a logit, when most others are done.  151936
// logits, fp16, device: one row, top-k 50 and top-p 0.95: 12.5 us; the largest: 4.1;
// 64 rows, the same: 20 and 7.0; 256 rows of spread-out logits, all of them: 87 us
// (reading them: 12; 28.7 M warp instructions: 25), and 52 where the given numbers
// leave no row to fp64 (64 rows: 38 and 18); 64 such rows under top-p alone, 50000
// tokens kept: 104.
#pragma once

#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "ql_common.cuh"

namespace ql {
namespace smp {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCtas = 16;         // of a row: the largest cluster
constexpr int kCuts = 4;             // thresholds of a round
constexpr int kMine = 16;            // thresholds of a round over the threads' largest logits
constexpr int kFew = 1024;           // tokens that one CTA sorts
constexpr int kFewer = kThreads / 4; // and those that it only compares with one another
constexpr double kOff = 6e-7;        // what sums of fp32 weights may be off, of themselves
constexpr int kBins = 4096;          // of a histogram
constexpr int kBlocks = 3 * kFew;    // a row's part has no more than these runs of the warps
constexpr int kStaged = 72 * 1024;   // bytes of a part that shared memory takes, two CTAs an SM

struct Params {
  const void* logits;                // [rows][stride]
  const float* uniform;              // [rows]
  const float *temperature, *top_p, *min_p;   // [rows], or null: the values for all below
  const int* top_k;
  long long* ids;                    // [rows]
  float* logprobs;                   // [rows] or null
  double temperature_all, top_p_all, min_p_all;
  long long top_k_all, stride;
  int rows, vocab, vec;              // vec: rows begin on 16 bytes
};

// How a type's values lie in order: as whole numbers, and back.  -0 comes as +0.
template <typename T> struct Type;
template <> struct Type<__half> {
  static constexpr int kLanes = 8;
  static __device__ __forceinline__ void decode(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = h2_to_f2(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ long long order(float x) {
    const unsigned b = __half_as_ushort(__float2half_rn(x));
    return b & 0x8000u ? 0xFFFFu ^ b : b | 0x8000u;
  }
  static __device__ __forceinline__ float value(long long k) {
    const unsigned b = (unsigned)k;
    return __half2float(__ushort_as_half((unsigned short)(b & 0x8000u ? b ^ 0x8000u : 0xFFFFu ^ b)));
  }
  static __device__ __forceinline__ float lowest() { return -65504.f; }
};
template <> struct Type<__nv_bfloat16> {
  static constexpr int kLanes = 8;
  static __device__ __forceinline__ void decode(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ long long order(float x) {
    const unsigned b = __float_as_uint(x) >> 16;
    return b & 0x8000u ? 0xFFFFu ^ b : b | 0x8000u;
  }
  static __device__ __forceinline__ float value(long long k) {
    const unsigned b = (unsigned)k;
    return __uint_as_float((b & 0x8000u ? b ^ 0x8000u : 0xFFFFu ^ b) << 16);
  }
  static __device__ __forceinline__ float lowest() { return __uint_as_float(0xFF7F0000u); }
};
template <> struct Type<float> {
  static constexpr int kLanes = 4;
  static __device__ __forceinline__ void decode(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ long long order(float x) {
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? 0xFFFFFFFFu ^ b : b | 0x80000000u;
  }
  static __device__ __forceinline__ float value(long long k) {
    const unsigned b = (unsigned)k;
    return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : 0xFFFFFFFFu ^ b);
  }
  static __device__ __forceinline__ float lowest() { return __uint_as_float(0xFF7FFFFFu); }
};

__device__ __forceinline__ void st_dsmem_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ __forceinline__ void st_dsmem_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_dsmem_u64(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_dsmem_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t atom_dsmem_add(uint32_t addr, uint32_t v) {
  uint32_t old;
  asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
  return old;
}

__device__ __forceinline__ unsigned order_of(float x) { return (unsigned)Type<float>::order(x); }
__device__ __forceinline__ float value_of(unsigned k) { return Type<float>::value(k); }

// 2^(i / 16).  In shared memory, where 16 of them take each bank once: lanes never wait for one another.
__constant__ const double kRoots[16] = {1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721,
                                        1.241857812073484, 1.2968395546510096, 1.3542555469368927, 1.4142135623730951,
                                        1.4768261459394993, 1.5422108254079407, 1.6104903319492543, 1.681792830507429,
                                        1.7562521603732995, 1.8340080864093424, 1.9152065613971474};
__shared__ double roots[16];

// A row's weights.  In fp32, with a = (x - top) log2(e) / T: 2^a from a whole number n near a, and 2^(a - n).  a - n is taken
// of the unrounded product: x hi - (n + base) in one rounding, n + base being exact, plus x lo; what base leaves of top's
// share is a factor on all of them, which sums get.  Weights end at 2^-100.  How far sums may be off, of themselves:
//   2^-22     each 2^(a - n), by ex2.approx
//   2^-24.5   a - n's two roundings
//   2^-22.4   eight of them added in pairs in fp32 (fp64 from there)
// together 4.6e-7; kOff is 6e-7.
struct Weights {
  float top, end;                    // the largest logit; where weights end
  float hi, lo, bias, base;          // log2(e) / T in two parts; 1.5 * 2^23 less top's share as a whole number; that share
  float zero;                        // where fp64 weights end: e^-700
  double factor;                     // on sums
  double inv_t, scale, share, high;  // 1 / T, log2(e) / T, top's share, top in fp64

  __device__ __forceinline__ void set_heat(double heat) {
    inv_t = 1.0 / heat;
    scale = inv_t * 1.4426950408889634074;
    hi = (float)fmin(scale, 1e37);                            // (no infinity, of which nothing could be taken 0 times)
    lo = (float)(scale - (double)hi);
  }
  __device__ __forceinline__ void set_top(float largest, double heat) {
    if (largest == INFINITY) hi = lo = 0.f, scale = inv_t = 0.0;          // the infinite ones alone, alike
    top = largest;
    share = largest == INFINITY ? 0.0 : (double)top * scale;
    high = in64(top);
    zero = fmaxf((float)((double)top - 700.0 * heat), -3.402823466e38f);
    end = fmaxf((float)((double)top - 69.314718 * heat), -3.402823466e38f);
    bias = 12582912.f - (float)rint(share);
    // a multiple of so small a power of two as lets whole numbers be added exactly
    const int e = max((__double2hiint(share) >> 20 & 0x7FF) - 1023, 7) - 21;      // (they are below 2^7)
    const double up = __hiloint2double((1023 - e) << 20, 0), grid = __hiloint2double((1023 + e) << 20, 0);
    base = (float)(rint(share * up) * grid);
    factor = exp2((double)base - share);
  }
  // whether fp32 will do
  __device__ __forceinline__ bool fine() const { return fabs(share) < 0x1p20 && scale < 0x1p40 && scale > 0x1p-40 && top < INFINITY; }

  __device__ __forceinline__ void two(float x, float y, float& v, float& w) const {
    const F2 m = fma2({x, y}, {hi, hi}, {bias, bias});
    const F2 s = add2(fma2(m, {-1.f, -1.f}, {12582912.f, 12582912.f}), {-base, -base});
    const F2 r = fma2({x, y}, {lo, lo}, fma2({x, y}, {hi, hi}, s));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v) : "f"(r.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(r.y));
    v = x >= end ? __int_as_float(__float_as_int(v) + (__float_as_int(m.x) << 23)) : 0.f;      // 0 of a NaN
    w = y >= end ? __int_as_float(__float_as_int(w) + (__float_as_int(m.y) << 23)) : 0.f;
  }
  __device__ __forceinline__ float one(float x) const {
    float v, w;
    two(x, x, v, w);
    return v;
  }
  // In fp64, some 40 instructions: of (x - top) as it is, 16 a as a whole number m (from fp32)
  // and a rest r; 2^(m / 16) from a table of 16 and the exponent, 2^(r / 16) by its Chebyshev expansion up to the fifth power
  // (2^-46; 1 of the largest, so that its ties are counted by whole numbers).  Numbers become fp64 by their bits: the
  // conversion's own instruction has a quarter of the rate.  (Numbers below fp32's normal ones, and 0, come out as one of
  // their size: 2^-126 of a logit.)
  __device__ __forceinline__ static double in64(float x) {
    const unsigned b = __float_as_uint(x);
    return __hiloint2double((int)(((b & 0x7FFFFFFFu) >> 3) + (896u << 20) | (b & 0x80000000u)), (int)(b << 29));
  }
  __device__ __forceinline__ double wide(float x) const {
    const float m = fmaf(fmaxf(x - top, -3.402823466e38f), 16.f * hi, 12582912.f);       // infinity less itself: a number
    const double r = fma(in64(x) - high, 16.0 * scale, -in64(m - 12582912.f));
    double y = 1.2716120543908984e-09;
    y = fma(y, r, 1.4676444622018903e-07);
    y = fma(y, r, 1.355080777639003e-05);
    y = fma(y, r, 0.0009383847924862057);
    y = fma(y, r, 0.04332169878499668);
    y = fma(y, r, 1.0) * roots[__float_as_int(m) & 15];
    return x >= zero ? __hiloint2double(__double2hiint(y) + (__float_as_int(m) - 0x4B400000 >> 4 << 20), __double2loint(y)) : 0.0;
  }
  // log(w / sum) of the weight of x: the sum's by its exponent, and the rest, 2/3 .. 4/3, in fp32 (2^-24 of at most 0.41)
  __device__ __forceinline__ float log_chance(float x, double sum) const {
    const int e = (__double2hiint(sum) + 0x000AAAAB >> 20) - 1023;
    const float rest = (float)__hiloint2double(__double2hiint(sum) - (e << 20), __double2loint(sum));
    return (float)((inv_t > 0.0 ? ((double)x - (double)top) * inv_t : 0.0) - ((double)logf(rest) + e * 0.69314718055994530942));
  }
};

// What a row's CTAs hold and send one another.  A meeting is a barrier of all of them (Row::meet); no store to another CTA
// comes before all have started.  What keeps one use from the next:
//   box    all_sum, all_u32, bound, locate, narrow send to a half, meet, read it; the other half is next (`turn`).
//   part   written, __syncthreads, read; then the call's meeting, or in the first CTA's own steps (cta_count, finish) a
//          __syncthreads before the next writing.  scan, sums alike.
//   block  locate: each CTA its own, read by itself before and behind the call's meeting; a meeting follows each call.
//   bins   narrow: each CTA adds to its own; a meeting; all read all CTAs' (twice); a meeting.
//   few    collect: all CTAs store keys in the first one's; a meeting; then the first CTA alone (finish, last_kept), until the
//          meeting behind that.
// So whoever begins with one member of the union comes from a meeting behind which nobody touches another.
//   found, here, at   collect: the CTA's own, here one for each call; its meeting follows.  count: added to by all CTAs, read
//          behind that meeting, before the next one.
//   edge, index, unsure, bin_*, mass_above, units_*   sent by one thread before a meeting, read behind it.
struct Shared {
  // What the cluster's CTAs have sent, in turn: a meeting's values to one half, the next one's to the other.  A CTA writes a
  // half again only behind the meeting in between, at which all have read what it held.  Sums and counts share the halves, of
  // which each is a union of its own: halves of different sizes in one union would lie over each other.
  union {
    double f64[kMaxCtas][kCuts];
    uint32_t u32[kMaxCtas][kMine];
  } box[2];
  union {
    double f64[kWarps][kCuts];
    uint32_t u32[kWarps][kMine];
  } part;
  union {
    double block[kBlocks];           // of many tokens: sums by runs of the warps
    unsigned bins[kBins];
    struct {                         // of few, in the cluster's first CTA
      unsigned long long key[kFew];
      unsigned long long weight[kFew], upto[kFew];      // in units of 2^-52 of the largest weight
    } few;
  };
  Weights weights;
  double before;
  unsigned long long scan[kWarps], sums[kWarps][2];
  unsigned long long found[kFew];    // tokens that this CTA has collected
  unsigned here[3], at, count[3];    // their number, their place in the first CTA's list; the list's length
  int run, index, unsure;
  float edge;
  // where a histogram's running sum crosses a target: its bins just below and just above that, -1 for none; what lies above
  // the one and up to the other
  int bin_above, bin_below;
  unsigned long long mass_above, units_above, units_below;
};

__shared__ Shared sh;                // not an argument: a function that gets it as one reads it by generic addresses

enum Kind { kCount, kMass, kExact }; // of a measure: the number of tokens, their weights in fp32, in fp64

// What a CTA has of a row: the tokens first .. first + count - 1 at src, in 16-byte runs, of which thread t takes t,
// t + kThreads ..; and its place in the cluster.
template <typename T>
struct Row {
  static constexpr int kLanes = Type<T>::kLanes;
  const T* src;
  int first, count, passes, rank, ctas;
  float mine;                        // this thread's largest logit
  bool vec;                          // runs are whole and aligned

  __device__ __forceinline__ uint4 load(int v, int thread) const {
    const int o = (v * kThreads + thread) * kLanes;
    if (vec && o + kLanes <= count) return *reinterpret_cast<const uint4*>(src + o);
    uint4 r;
    T* e = reinterpret_cast<T*>(&r);
    #pragma unroll
    for (int i = 0; i < kLanes; ++i) e[i] = o + i < count ? src[o + i] : (T)(-INFINITY);
    return r;
  }
  __device__ __forceinline__ uint4 load(int v) const { return load(v, (int)threadIdx.x); }
  // f(run, its values), one run after another: the code comes from memory, 128 bytes some 100 cycles, and mostly runs a few
  // times over shared memory.  (Four runs a turn: 33.4 rather than 29.1 us for 37 rows of 32003, 35.8 rather than 30.5 for 64
  // of 128256; with two on their way 30.1 and 31.6.)
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    #pragma unroll 1
    for (int v = 0; v < passes; ++v) {
      float x[kLanes];
      Type<T>::decode(load(v), x);
      f(v, x);
    }
  }
  __device__ __forceinline__ int index(int v, int thread) const { return first + (v * kThreads + thread) * kLanes; }
  __device__ __forceinline__ int index(int v) const { return index(v, (int)threadIdx.x); }
  // f(values, index of the first) of the runs of those threads whose `holds` is set.  Where they are few of a warp, its lanes
  // take these one thread after another, a run a lane.
  template <typename F>
  __device__ __forceinline__ void each_of(bool holds, F f) const {
    unsigned holders = __ballot_sync(0xffffffffu, holds);
    if (__popc(holders) * ((passes + 31) / 32) < passes) {
      for (; holders; holders &= holders - 1) {
        const int thread = (int)(threadIdx.x & ~31u) + __ffs(holders) - 1;
        for (int v = threadIdx.x & 31; v < passes; v += 32) {
          float x[kLanes];
          Type<T>::decode(load(v, thread), x);
          f(x, index(v, thread));
        }
      }
    } else if (holds) {
      each([&](int v, const float (&x)[kLanes]) { f(x, index(v)); });
    }
  }
  __device__ __forceinline__ void meet() const {             // all threads of the cluster
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
  }
};

// ------------------------------------------------------- sums over the cluster
// A warp's sums of N values (N 1, 2 or 4) with the fewest exchanges: of value i in the lanes 32 / N i .. 32 / N (i + 1) - 1.
template <int N>
__device__ __forceinline__ double warp_sums(const double (&v)[N]) {
  const int lane = threadIdx.x & 31;
  double a = v[0];
  if constexpr (N == 4) {
    const bool up = lane & 16, high = lane & 8;
    const double b0 = __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], 16), b1 = __shfl_xor_sync(0xffffffffu, up ? v[1] : v[3], 16);
    const double c0 = (up ? v[2] : v[0]) + b0, c1 = (up ? v[3] : v[1]) + b1;
    a = (high ? c1 : c0) + __shfl_xor_sync(0xffffffffu, high ? c0 : c1, 8);
  } else if constexpr (N == 2) {
    const bool up = lane & 16;
    a = (up ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, up ? v[0] : v[1], 16);
  }
  #pragma unroll
  for (int o = 16 / N; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  return a;
}
// The same in all threads.
template <typename T, int N>
__device__ __forceinline__ void all_sum(const Row<T>& row, int& turn, double (&v)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = lane * N / 32;
  double s = warp_sums<N>(v);
  if (lane % (32 / N) == 0) sh.part.f64[warp][i] = s;
  __syncthreads();
  turn ^= 1;
  if (warp == 0) {
    double w[N];
    #pragma unroll
    for (int q = 0; q < N; ++q) w[q] = lane < kWarps ? sh.part.f64[lane][q] : 0.0;
    s = warp_sums<N>(w);
    #pragma unroll
    for (int q = 0; q < N; ++q) {
      const double all = __shfl_sync(0xffffffffu, s, q * (32 / N));
      if (lane < row.ctas) st_dsmem_f64(dsmem_addr(smem_u32(&sh.box[turn].f64[row.rank][q]), (uint32_t)lane), all);
    }
  }
  row.meet();
  double w[N];
  #pragma unroll
  for (int q = 0; q < N; ++q) w[q] = lane < row.ctas ? sh.box[turn].f64[lane][q] : 0.0;
  s = warp_sums<N>(w);
  #pragma unroll
  for (int q = 0; q < N; ++q) v[q] = __shfl_sync(0xffffffffu, s, q * (32 / N));
}
// `op` of a warp's 32 values, the same in all its lanes; `none` changes nothing.
template <typename T, int N, typename Op>
__device__ __forceinline__ void all_u32(const Row<T>& row, int& turn, uint32_t (&v)[N], uint32_t none, Op op) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  #pragma unroll
  for (int i = 0; i < N; ++i) v[i] = op(v[i]);
  if (lane == 0)
    #pragma unroll
    for (int i = 0; i < N; ++i) sh.part.u32[warp][i] = v[i];
  __syncthreads();
  turn ^= 1;
  if (warp == 0) {
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t s = op(lane < kWarps ? sh.part.u32[lane][i] : none);
      if (lane < row.ctas) st_dsmem_u32(dsmem_addr(smem_u32(&sh.box[turn].u32[row.rank][i]), (uint32_t)lane), s);
    }
  }
  row.meet();
  #pragma unroll
  for (int i = 0; i < N; ++i) v[i] = op(lane < row.ctas ? sh.box[turn].u32[lane][i] : none);
}
// F at thresholds: the number of tokens x >= cut (not of a NaN), or the sum of their weights.  A function of its own for
// each kind: the code is read from memory once a launch, and that is a good part of a short row's time.
template <typename T, Kind KIND, int N>
__device__ __noinline__ double4 measure_of(const Row<T> row, int& turn, float4 at) {
  constexpr int kLanes = Type<T>::kLanes;
  const float cut[kCuts] = {at.x, at.y, at.z, at.w};
  const Weights w = sh.weights;
  double f[N] = {};
  if constexpr (KIND == kCount) {
    uint32_t n[N] = {};
    row.each([&](int, const float (&x)[kLanes]) {
      #pragma unroll
      for (int e = 0; e < kLanes; ++e)
        #pragma unroll
        for (int i = 0; i < N; ++i) n[i] += x[e] >= cut[i];
    });
    all_u32<T, N>(row, turn, n, 0u, [](uint32_t v) { return __reduce_add_sync(0xffffffffu, v); });
    return make_double4((double)n[0], (double)n[1], N > 2 ? (double)n[N - 2] : 0.0, N > 2 ? (double)n[N - 1] : 0.0);
  } else {
    row.each([&](int, const float (&x)[kLanes]) {
      if constexpr (KIND == kMass) {
        float s[2][N] = {};
        #pragma unroll
        for (int e = 0; e < kLanes; e += 2) {
          float v[2];
          w.two(x[e], x[e + 1], v[0], v[1]);
          #pragma unroll
          for (int i = 0; i < N; ++i)
            #pragma unroll
            for (int q = 0; q < 2; ++q)
              if (x[e + q] >= cut[i]) s[q][i] += v[q];
        }
        #pragma unroll
        for (int i = 0; i < N; ++i) f[i] += (double)(s[0][i] + s[1][i]);
      } else {
        #pragma unroll
        for (int e = 0; e < kLanes; ++e) {
          const double v = w.wide(x[e]);
          #pragma unroll
          for (int i = 0; i < N; ++i) f[i] += x[e] >= cut[i] ? v : 0.0;
        }
      }
    });
    all_sum<T, N>(row, turn, f);
    const double by = KIND == kMass ? w.factor : 1.0;
    return make_double4(f[0] * by, f[1] * by, N > 2 ? f[N - 2] * by : 0.0, N > 2 ? f[N - 1] * by : 0.0);
  }
}
template <typename T, Kind KIND>
__device__ __forceinline__ double4 measure(const Row<T>& row, int& turn, float4 at) {
  return measure_of<T, KIND, kCuts>(row, turn, at);
}
template <typename T, Kind KIND>
__device__ __forceinline__ double2 measure(const Row<T>& row, int& turn, float2 at) {
  const double4 f = measure_of<T, KIND, 2>(row, turn, make_float4(at.x, at.y, NAN, NAN));
  return make_double2(f.x, f.y);
}

// The largest value whose F reaches `target`, from F(from) >= target on; *above: F of what lies above it.
template <typename T, Kind KIND>
__device__ __forceinline__ float search(const Row<T>& row, int& turn, float from, double target, double* above) {
  long long lo = Type<T>::order(from), hi = Type<T>::order(sh.weights.top) + 1;
  *above = 0.0;
  while (hi - lo > 1) {
    long long at[kCuts];
    #pragma unroll
    for (int i = 0; i < kCuts; ++i) at[i] = lo + max((hi - lo) * (i + 1) / (kCuts + 1), 1ll);
    const double4 g = measure<T, KIND>(row, turn, make_float4(Type<T>::value(at[0]), Type<T>::value(at[1]),
                                                                  Type<T>::value(at[2]), Type<T>::value(at[3])));
    const double f[kCuts] = {g.x, g.y, g.z, g.w};
    #pragma unroll
    for (int i = 0; i < kCuts; ++i) {
      if (f[i] >= target) {
        lo = max(lo, at[i]);
      } else if (at[i] < hi) {
        hi = at[i];
        *above = f[i];
      }
    }
  }
  return Type<T>::value(lo);
}

// A value v such that the threads' largest logits >= v number `target`, or weigh as much: not the largest such, but one
// with few of them above it.  False: there is none.  Lane i looks after threshold i.
template <typename T>
__device__ __noinline__ bool bound(const Row<T> row, int& turn, bool mass, float least, double target, float* v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float top = sh.weights.top;
  constexpr double kUnit = 0x1p22;                            // weights are counted in whole units: never too much
  const uint32_t unit = mass ? (uint32_t)((double)sh.weights.one(row.mine) * (sh.weights.factor * kUnit)) : 1u;
  const double wanted = mass ? target * kUnit : target, enough_of = mass ? wanted * 1.02 : wanted * 1.25 + 16.0;
  long long lo = Type<T>::order(least), hi = Type<T>::order(top) + 1;
  bool found = false;
  #pragma unroll 1
  for (int round = 0; round < 10; ++round) {
    // even in value, where the values are that near; else even in their order
    const float from = Type<T>::value(lo), span = Type<T>::value(hi) - from;
    long long at = lo + (hi - lo) * (lane & (kMine - 1)) / kMine;
    if (span < 1024.f) at = min(max(Type<T>::order(fmaf(span, (float)(lane & (kMine - 1)) / kMine, from) + 0.f), lo), hi - 1);
    const float cut = Type<T>::value(at);
    uint32_t f = 0;
    if (mass) {
      #pragma unroll 4
      for (int i = 0; i < kMine; ++i) {
        const uint32_t n = __reduce_add_sync(0xffffffffu, row.mine >= __shfl_sync(0xffffffffu, cut, i) ? unit : 0u);
        if (lane == i) f = n;
      }
    } else {
      #pragma unroll 4
      for (int i = 0; i < kMine; ++i) {
        const uint32_t n = __popc(__ballot_sync(0xffffffffu, row.mine >= __shfl_sync(0xffffffffu, cut, i)));
        if (lane == i) f = n;
      }
    }
    if (lane < kMine) sh.part.u32[warp][lane] = f;
    __syncthreads();
    turn ^= 1;
    if (warp == 0 && lane < kMine) {
      f = 0;
      #pragma unroll
      for (int w = 0; w < kWarps; ++w) f += sh.part.u32[w][lane];
      #pragma unroll
      for (int r = 0; r < kMaxCtas; ++r)
        if (r < row.ctas) st_dsmem_u32(dsmem_addr(smem_u32(&sh.box[turn].u32[row.rank][lane]), (uint32_t)r), f);
    }
    row.meet();
    unsigned long long sum = 0;
    #pragma unroll
    for (int r = 0; r < kMaxCtas; ++r) sum += r < row.ctas ? sh.box[turn].u32[r][lane & (kMine - 1)] : 0u;
    double all = (double)sum;
    const unsigned enough = __ballot_sync(0xffffffffu, lane < kMine && all >= wanted);
    if (!found && !(enough & 1u)) return false;
    found = true;                                             // of lo, and so of some threshold
    const int pick = 31 - __clz(enough | 1u);
    const long long next = __shfl_sync(0xffffffffu, at, (pick + 1) & (kMine - 1));
    if (pick + 1 < kMine) hi = next;
    lo = __shfl_sync(0xffffffffu, at, pick);
    all = __shfl_sync(0xffffffffu, all, pick);
    // (weights: what lies within 2^(1/32) of the last is not told apart, however few are above)
    if (hi - lo <= 1 || all <= enough_of || (mass && (double)(Type<T>::value(hi) - Type<T>::value(lo)) * sh.weights.scale < 0.03125)) break;
  }
  *v = Type<T>::value(lo);
  return true;
}

// ------------------------------------------------------------ many are kept
// The first token, by index, at which the running sum of what it counts exceeds a target, or the last that counts.  kCount:
// the tokens equal to `edge`, and the target is `wanted`.  Else the weights of those above `edge`, and of those equal to it
// up to index `last`, and the target is `wanted` of their sum.  found(index, x, sum) in one thread of the cluster; the sum is
// returned.  kMass: where a running sum comes too close to the target to tell, sh.unsure is set in all CTAs, to be read
// behind the next meeting.
template <typename T, Kind KIND, typename Found>
__device__ __forceinline__ double locate(const Row<T>& row, int& turn, float edge, int last, double wanted, Found found) {
  constexpr int kLanes = Type<T>::kLanes;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Weights weights = sh.weights;
  weights.end = fmaxf(weights.end, edge);                     // weights below the edge are 0
  weights.zero = fmaxf(weights.zero, edge);
  const bool whole = last == 0x7FFFFFFF;                      // all that equal `edge`
  auto counts = [&](float x, int i) { return !(x == edge && i > last); };
  // a block: a run of a warp; four at a time, whose sums go through the warp together
  #pragma unroll 1
  for (int v = 0; v < row.passes; v += 4) {
    uint4 r[4];
    #pragma unroll
    for (int q = 0; q < 4; ++q)
      if (v + q < row.passes) r[q] = row.load(v + q);
    double s[4] = {};
    #pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (v + q >= row.passes) continue;
      float x[kLanes];
      Type<T>::decode(r[q], x);
      if constexpr (KIND == kCount) {
        int n = 0;
        #pragma unroll
        for (int e = 0; e < kLanes; ++e) n += x[e] == edge;
        s[q] = n;
      } else if constexpr (KIND == kMass) {
        float p[kLanes];
        #pragma unroll
        for (int e = 0; e < kLanes; e += 2) weights.two(x[e], x[e + 1], p[e], p[e + 1]);
        if (!whole)
          #pragma unroll
          for (int e = 0; e < kLanes; ++e)
            if (!counts(x[e], row.index(v + q) + e)) p[e] = 0.f;
        #pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1)
          #pragma unroll
          for (int e = 0; e < o; ++e) p[e] += p[e + o];
        s[q] = p[0];
      } else {
        #pragma unroll
        for (int e = 0; e < kLanes; ++e) s[q] += whole || counts(x[e], row.index(v + q) + e) ? weights.wide(x[e]) : 0.0;
      }
    }
    const double all = warp_sums<4>(s);
    if (lane % 8 == 0 && v + lane / 8 < row.passes) sh.block[(v + lane / 8) * kWarps + warp] = all;
  }
  __syncthreads();
  turn ^= 1;
  const int blocks = row.passes * kWarps, per_lane = (blocks + 31) / 32;
  auto upto_lane = [&](double v) {
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  // what lies before a lane, of sums up to it: not those less its own, of which a weight of 1 leaves nothing below 2^-53
  auto before_lane = [&](double to) {
    const double b = __shfl_up_sync(0xffffffffu, to, 1);
    return lane > 0 ? b : 0.0;
  };
  double own = 0.0, upto = 0.0;
  if (warp == 0) {
    for (int i = 0; i < per_lane; ++i)
      if (lane * per_lane + i < blocks) own += sh.block[lane * per_lane + i];
    upto = upto_lane(own);
    const double all = __shfl_sync(0xffffffffu, upto, 31);
    if (lane < row.ctas) st_dsmem_f64(dsmem_addr(smem_u32(&sh.box[turn].f64[row.rank][0]), (uint32_t)lane), all);
  }
  row.meet();
  // each warp finds whose part holds the token, by the same sums: first lanes, CTAs; then, in that CTA, lanes' blocks
  const double part = lane < row.ctas ? sh.box[turn].f64[lane][0] : 0.0;
  double to = upto_lane(part);
  const double sum = __shfl_sync(0xffffffffu, to, 31), t = KIND == kCount ? wanted : wanted * sum;
  auto pick = [&](bool some, bool past) {                     // the first past the target, else the last that has some
    const unsigned any = __ballot_sync(0xffffffffu, some), over = __ballot_sync(0xffffffffu, some && past);
    return over ? __ffs(over) - 1 : 31 - __clz(any);
  };
  const int owner = pick(part > 0.0, to > t);
  if (owner == row.rank) {
    double before = __shfl_sync(0xffffffffu, before_lane(to), owner);
    if (warp == 0) {
      const int at_lane = pick(own > 0.0, before + upto > t);
      const double lanes = before_lane(upto);
      if (lane == at_lane) {
        double run = before + lanes, kept = run;
        int at = 0;
        for (int i = lane * per_lane; i < min((lane + 1) * per_lane, blocks); ++i) {
          const double w = sh.block[i];
          if (w > 0.0) {
            at = i;
            kept = run;
            if (run + w > t) break;
          }
          run += w;
        }
        sh.run = at;
        sh.before = kept;
      }
    }
    __syncthreads();
    if (warp == sh.run % kWarps) {
      const int v = sh.run / kWarps;
      before = sh.before;
      float x[kLanes];
      double w[kLanes], s = 0.0;
      Type<T>::decode(row.load(v), x);
      #pragma unroll
      for (int e = 0; e < kLanes; ++e) {
        const int i = row.index(v) + e;
        w[e] = KIND == kCount ? (double)(x[e] == edge) : !counts(x[e], i) ? 0.0 : KIND == kMass ? (double)weights.one(x[e]) : weights.wide(x[e]);
        s += w[e];
      }
      to = upto_lane(s);
      const int at_lane = pick(s > 0.0, before + to > t);
      const double lanes = before_lane(to);
      if (lane == at_lane) {
        double run = before + lanes, from = run, until = run;
        float x_pick = x[0];
        int e_pick = 0;
        bool done = false;
        #pragma unroll
        for (int e = 0; e < kLanes; ++e) {
          if (w[e] > 0.0 && !done) {
            e_pick = e;
            x_pick = x[e];
            from = run;
            until = run + w[e];
            done = until > t;
          }
          run += w[e];
        }
        if (KIND == kMass && (t - from <= 2.0 * kOff * t || until - t <= 2.0 * kOff * t))
          for (int r = 0; r < row.ctas; ++r) st_dsmem_u32(dsmem_addr(smem_u32(&sh.unsure), (uint32_t)r), 1u);
        found(row.index(v) + e_pick, x_pick, sum);
      }
    }
  }
  return sum;
}
template <typename T, Kind KIND>
__device__ __noinline__ void draw(const Row<T> row, int& turn, float edge, int last, double u, long long* id, float* logprob) {
  locate<T, KIND>(row, turn, edge, last, u, [&](int i, float x, double sum) {
    *id = i;
    if (logprob) *logprob = sh.weights.log_chance(x, sum * (KIND == kMass ? sh.weights.factor : 1.0));
  });
  row.meet();
}

// ------------------------------------------------------------- few are kept
// The tokens cut <= x < below, as (value, index) in the cluster's first CTA; how many there are (past kFew the list is cut
// off).  `call`: 0, 1, 2, another for each call of a row.
template <typename T>
__device__ __noinline__ unsigned collect(const Row<T> row, int call, float cut, float below) {
  constexpr int kLanes = Type<T>::kLanes;
  auto take = [&](const float (&x)[kLanes], int index) {
    unsigned some = 0;
    #pragma unroll
    for (int e = 0; e < kLanes; ++e) some |= (x[e] >= cut && !(x[e] >= below)) << e;
    if (some == 0) return;
    unsigned at = atomicAdd(&sh.here[call], (unsigned)__popc(some));
    #pragma unroll
    for (int e = 0; e < kLanes; ++e)
      if (some >> e & 1) {
        if (at < kFew) sh.found[at] = (unsigned long long)order_of(x[e] + 0.f) << 32 | (0xFFFFFFFFu - (unsigned)(index + e));
        ++at;
      }
  };
  row.each_of(row.mine >= cut, take);
  __syncthreads();
  const unsigned here = sh.here[call];
  const uint32_t counter = dsmem_addr(smem_u32(&sh.count[call]), 0), keys = dsmem_addr(smem_u32(&sh.few.key[0]), 0);
  if (here > 0) {
    if (threadIdx.x == 0) sh.at = atom_dsmem_add(counter, here);
    __syncthreads();
    for (unsigned i = threadIdx.x; i < here && sh.at + i < kFew; i += kThreads) st_dsmem_u64(keys + (sh.at + i) * 8u, sh.found[i]);
  }
  row.meet();
  return ld_dsmem_u32(counter);
}

// Sums over the first CTA, the same in all its threads.
__device__ __forceinline__ unsigned cta_count(unsigned n) {
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.part.u32[threadIdx.x >> 5][0] = n;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, (threadIdx.x & 31) < kWarps ? sh.part.u32[threadIdx.x & 31][0] : 0u);
}
__device__ __forceinline__ unsigned long long warp_whole(unsigned long long v) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ unsigned long long cta_sum(unsigned long long v) {
  v = warp_whole(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.scan[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_whole((threadIdx.x & 31) < kWarps ? sh.scan[threadIdx.x & 31] : 0ull);
}
__device__ __forceinline__ int index_of(unsigned long long key) { return (int)(0xFFFFFFFFu - (unsigned)key); }

// Sorts key[0 .. n) from the largest down, n <= kFew; upto is lost.  A bitonic network over registers, one key a thread, two
// above kThreads: partners within a warp exchange by shuffles, others through upto and key in turn, one barrier a step.  200
// keys take 3900 cycles, 1024 12800; all steps in shared memory, with a barrier each, took 11700 and 18000.
template <int J>
__device__ __forceinline__ void exchange(unsigned long long& v, bool larger) {
  const unsigned long long other = __shfl_xor_sync(0xffffffffu, v, J);
  v = (larger == ((threadIdx.x & J) == 0)) ? max(v, other) : min(v, other);
}
// the steps within a warp of blocks of k
template <int J>
__device__ __forceinline__ void exchanges(unsigned long long& v, unsigned index, unsigned k) {
  const bool larger = (index & k) == 0;
  if constexpr (J >= 16) exchange<16>(v, larger);
  if constexpr (J >= 8) exchange<8>(v, larger);
  if constexpr (J >= 4) exchange<4>(v, larger);
  if constexpr (J >= 2) exchange<2>(v, larger);
  exchange<1>(v, larger);
}
__device__ __noinline__ void sort(unsigned n) {
  const unsigned tid = threadIdx.x;
  unsigned size = 64;
  while (size < n) size *= 2;
  const bool live = tid < size, two = size > kThreads;
  __syncthreads();
  unsigned long long a = tid < n ? sh.few.key[tid] : 0, b = tid + kThreads < n ? sh.few.key[tid + kThreads] : 0;
  unsigned long long *at = sh.few.upto, *next = sh.few.key;
  auto first = [&](unsigned long long& v) {
    exchanges<1>(v, tid, 2);
    exchanges<2>(v, tid, 4);
    exchanges<4>(v, tid, 8);
    exchanges<8>(v, tid, 16);
    exchanges<16>(v, tid, 32);
  };
  if (live) first(a);
  if (two) first(b);
  #pragma unroll 1
  for (unsigned k = 64; k <= size; k *= 2) {
    #pragma unroll 1
    for (unsigned j = k / 2; j >= 32; j /= 2) {
      if (j == kThreads) {
        const unsigned long long most = max(a, b);
        b = min(a, b);
        a = most;
        continue;
      }
      if (live) at[tid] = a;
      if (two) at[tid + kThreads] = b;
      __syncthreads();
      const bool low = (tid & j) == 0;
      if (live) {
        const unsigned long long other = at[tid ^ j];
        a = low == ((tid & k) == 0) ? max(a, other) : min(a, other);
      }
      if (two) {
        const unsigned long long other = at[(tid ^ j) + kThreads];
        b = low == ((tid + kThreads & k) == 0) ? max(b, other) : min(b, other);
      }
      unsigned long long* swap = at;
      at = next;
      next = swap;
    }
    if (live) exchanges<16>(a, tid, k);
    if (two) exchanges<16>(b, tid + kThreads, k);
  }
  __syncthreads();
  if (live) sh.few.key[tid] = a;
  if (two) sh.few.key[tid + kThreads] = b;
  __syncthreads();
}
// Running sums of weight[0 .. n) to upto[0 .. n).
__device__ __noinline__ void run_up(unsigned n) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned i = 2 * threadIdx.x;
  const unsigned long long a = i < n ? sh.few.weight[i] : 0, b = i + 1 < n ? sh.few.weight[i + 1] : 0;
  unsigned long long s = a + b;
  #pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) sh.scan[warp] = s;
  __syncthreads();
  const unsigned long long before = warp_whole(lane < warp ? sh.scan[lane] : 0ull);
  if (i < n) sh.few.upto[i] = before + (s - b);
  if (i + 1 < n) sh.few.upto[i + 1] = before + s;
  __syncthreads();
}
// Weights of few tokens, as whole numbers: additions of these are exact and quick.  What is less than half a unit is nothing,
// as beside 1 in fp64 (lifted to a unit it would be drawn where u falls between two tokens to the bit).
constexpr double kWhole = 0x1p52;
__device__ __forceinline__ unsigned long long whole(double w, double per) { return __double2ull_rn(fmin(w * per, kWhole)); }
__device__ __noinline__ void weigh_few(unsigned n, int value_at = 32, double per = kWhole) {      // where keys have the value
  for (unsigned i = threadIdx.x; i < n; i += kThreads)
    sh.few.weight[i] = whole(sh.weights.wide(value_of((unsigned)(sh.few.key[i] >> value_at))), per);
  __syncthreads();
}
// How the token is drawn of the kept weights, whose sum is `total` units of 2^-52: in units of 1 / per, with t of them the
// target.  From u = 2^-12 on they are the same units, whose rounding is 2^-31 of the target at most (half a unit of 1024
// tokens).  Below, small weights come to matter: units so fine that the target is 2^51 of them, larger weights than it cut off
// at 2^52.  At the ends each token that has a weight counts, however small: the first is drawn, or the last.
struct Draw {
  double per;
  unsigned long long t;
  bool same;
};
__device__ __forceinline__ Draw draw_of(double u, unsigned long long total) {
  if (u >= 0x1p-12 && u < 1.0) {     // u is fp32: whole in units of 2^-36; the product to its last bit, so that ties are ties
    const unsigned long long m = (unsigned long long)(u * 0x1p36);
    return {kWhole, __umul64hi(m, total) << 28 | m * total >> 36, true};
  }
  if (u <= 0.0 || u >= 1.0) return {0x1p1023, u <= 0.0 ? 0ull : ~0ull, false};      // (weights end at e^-700)
  return {0x1p103 / (u * (double)total), 1ull << 51, false};
}

struct Filters {
  long long top_k;                   // 0: off
  double top_p;                      // 1: off
  float cut;                         // min-p's
};
// The rest, in the first CTA, of n weighted tokens that hold all that are kept (and, where top-k is on, all its tokens).
// `sum` is what top-p is of where top-k is off, right to `off` of itself.  False: it came too close to the weights before some
// token to tell whether that is kept; the list is as it was, or sorted.
//
// Up to kFewer tokens are not sorted: four or eight threads add up, for a token, the weights of those before it in the order,
// then, of those kept, the weights up to it by index.
__device__ __noinline__ bool finish(unsigned n, const Filters& filters, double sum, double off, double u, long long* id, float* logprob) {
  const unsigned tid = threadIdx.x;
  auto& key = sh.few.key;
  auto& weight = sh.few.weight;
  auto& upto = sh.few.upto;
  const bool k_on = filters.top_k > 0, p_on = filters.top_p < 1.0;
  const double top_p = fmax(filters.top_p, 0.0);
  const unsigned most = k_on && filters.top_k < (long long)n ? (unsigned)filters.top_k : n;
  double target = top_p * sum * kWhole, near = 2.0 * off * target;
  // what lies before a token comes to less than the target; too close to it to tell
  auto less = [&](unsigned long long before) { return !p_on || (double)before < target; };
  auto close = [&](unsigned long long before) { return p_on && off > 0.0 && fabs((double)before - target) <= near; };
  if (n <= kFewer) {
    const unsigned shift = n <= kFewer / 2 ? 3 : 2, i = tid >> shift, step = 1u << shift, lane = tid & (step - 1);
    const unsigned long long k = i < n ? key[i] : ~0ull, w = i < n ? weight[i] : 0;
    auto over_step = [&](auto v) {
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (shift == 3) v += __shfl_xor_sync(0xffffffffu, v, 4);
      return v;
    };
    unsigned rank = 0;
    unsigned long long before = 0;
    #pragma unroll 4
    for (unsigned j = lane; j < n; j += step) {
      const bool ahead = key[j] > k;
      rank += ahead;
      before += ahead ? weight[j] : 0;
    }
    rank = over_step(rank);
    before = over_step(before);
    const bool mine = lane == 0 && i < n;                     // one thread speaks for a token
    if (k_on && p_on) target = top_p * (double)cta_sum(mine && rank < most ? w : 0);
    const bool kept = i < n && (rank == 0 || (rank < most && less(before) && value_of((unsigned)(k >> 32)) >= filters.cut));
    if (mine) upto[i] = kept ? w : 0;
    if (__syncthreads_or(mine && rank > 0 && close(before))) return false;
    const unsigned long long total = cta_sum(mine && kept ? w : 0);
    const Draw draw = draw_of(u, total);
    unsigned long long share = w;                             // in the draw's units
    if (!draw.same) {
      share = i < n ? whole(sh.weights.wide(value_of((unsigned)(k >> 32))), draw.per) : 0;
      if (mine) upto[i] = kept ? share : 0;
      __syncthreads();
    }
    unsigned long long to = 0;
    #pragma unroll 4
    for (unsigned j = lane; j < n; j += step) to += (unsigned)key[j] >= (unsigned)k ? upto[j] : 0;     // ~index: those up to it
    to = over_step(to);
    // the first whose running sum passes t, else the last that has a weight
    const unsigned at = kept && share > 0 ? (unsigned)index_of(k) : 0xFFFFFFFFu;
    const unsigned past = __reduce_min_sync(0xffffffffu, to > draw.t ? at : 0xFFFFFFFFu);
    const unsigned end = __reduce_max_sync(0xffffffffu, at + 1);          // 0: none
    if ((tid & 31) == 0) {
      sh.part.u32[tid >> 5][0] = past;
      sh.part.u32[tid >> 5][1] = end;
    }
    __syncthreads();
    const unsigned pick_past = __reduce_min_sync(0xffffffffu, (tid & 31) < kWarps ? sh.part.u32[tid & 31][0] : 0xFFFFFFFFu);
    const unsigned pick_end = __reduce_max_sync(0xffffffffu, (tid & 31) < kWarps ? sh.part.u32[tid & 31][1] : 0u);
    const unsigned pick = pick_past != 0xFFFFFFFFu ? pick_past : pick_end - 1;
    if (mine && kept && at == pick) {
      *id = (long long)pick;
      if (logprob) *logprob = sh.weights.log_chance(value_of((unsigned)(k >> 32)), (double)total * (1.0 / kWhole));
    }
    return true;
  }
  sort(n);
  weigh_few(n);
  run_up(n);
  if (k_on) target = top_p * (double)upto[most - 1];
  bool unsure = false;
  unsigned kept = 0;
  for (unsigned i = 2 * tid; i < 2 * tid + 2 && i < most; ++i) {
    const unsigned long long before = i > 0 ? upto[i - 1] : 0;
    unsure |= i > 0 && close(before);
    kept += i == 0 || (less(before) && value_of((unsigned)(key[i] >> 32)) >= filters.cut);
  }
  if (__syncthreads_or(unsure)) return false;
  kept = cta_count(kept);
  const unsigned long long total = upto[kept - 1];
  const Draw draw = draw_of(u, total);
  for (unsigned i = tid; i < kept; i += kThreads) key[i] = key[i] << 32 | key[i] >> 32;       // by index
  __syncthreads();
  sort(kept);
  weigh_few(kept, 0, draw.per);
  run_up(kept);
  unsigned before = 0;
  for (unsigned i = 2 * tid; i < 2 * tid + 2 && i < kept; ++i) before += upto[i] <= draw.t;
  unsigned pick = cta_count(before);
  if (tid == 0) {
    if (pick >= kept) pick = kept - 1;
    while (pick > 0 && weight[pick] == 0) --pick;
    *id = index_of(key[pick] >> 32);
    if (logprob) *logprob = sh.weights.log_chance(value_of((unsigned)key[pick]), (double)total * (1.0 / kWhole));
  }
  return true;
}

// Narrows lo <= x < hi (as Type::order), where F crosses `target`, right to `margin`, by a histogram of these tokens' weights;
// *above: F(hi), in units of 2^-42 of the largest.  Returns no less than the number of tokens that are left, or infinity where
// that is not known.
//
// A bin is a step of 1 / per in log2 of the weight, and counts units of 2^-bits of the weight in its middle: 2^-t of a token's
// distance t from there, |t| <= 1/80, is 1 - t ln 2 + (t ln 2)^2 / 2 to 2^-23, so the units say both the weights and, to 1 in
// 100, the number, and take no ex2.  bits: as many as let 32 hold a CTA's tokens.  Bins are found by one rounding of a product and a difference, which never falls where x rises: each is a range of values.
constexpr double kPart = 0x1p42;
template <typename T>
__device__ __noinline__ double narrow(const Row<T> row, int& turn, double target, double margin, long long* lo, long long* hi,
                                      unsigned long long* above, int bits, bool wide) {
  constexpr int kLanes = Type<T>::kLanes;
  constexpr float kMagic = 12582912.f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float low = Type<T>::value(*lo), high = Type<T>::value(*hi);
  const double scale = sh.weights.scale, octaves = ((double)high - (double)low) * scale;
  // 32 octaves, below which few weights reach so far that top-p's target is there; less where less is left
  const double per = fmin(fmax((kBins - 1) / octaves, wide ? kBins / 32.0 : 0.0), 0x1p24);
  const float h = (float)(per * scale), off = (float)(per * scale * (double)high), one = (float)(1 << bits);
  const float slope = (float)(one * 0.6931471805599453 / per), curve = (float)(0.5 * 0.6931471805599453 * 0.6931471805599453 * one / (per * per));
  auto place = [&](float x) { return fmaxf(fmaf(x, -h, off), 0.f) + kMagic; };
  auto bin_of = [&](float place) { return __float_as_int(place) - 0x4B400000; };
  for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
  __syncthreads();
  if (threadIdx.x == 0) sh.bin_above = sh.bin_below = -1;
  row.each([&](int, const float (&x)[kLanes]) {
    #pragma unroll
    for (int e = 0; e < kLanes; ++e) {
      const float f = fmaxf(fmaf(x[e], -h, off), 0.f), m = f + kMagic, t = f - (m - kMagic);
      const float units = fmaf(t, fmaf(t, curve, -slope), one + kMagic);
      const int bin = bin_of(m);
      if (x[e] >= low && x[e] < high && bin < kBins) atomicAdd(&sh.bins[bin], (unsigned)(__float_as_int(units) - 0x4B400000));
    }
  });
  row.meet();
  // each CTA takes a run of the bins, each thread some of that
  const int each = kBins / row.ctas, run = max(each / kThreads, 1), first = row.rank * each + (int)threadIdx.x * run;
  const bool live = (int)threadIdx.x * run < each;
  auto units_of = [&](int bin) {
    unsigned long long u = 0;
    #pragma unroll
    for (int r = 0; r < kMaxCtas; ++r)                        // all on their way together
      if (r < row.ctas) u += ld_dsmem_u32(dsmem_addr(smem_u32(&sh.bins[bin]), (uint32_t)r));
    return u;
  };
  const float middle = (float)(((double)high - (double)sh.weights.top) * scale), step = (float)(1.0 / per);
  auto mass_of = [&](int bin, unsigned long long units) {
    return __double2ull_rn((double)units * (double)(exp2f(fmaf((float)bin, -step, middle)) * (float)kPart / one));
  };
  unsigned long long mass = 0, units = 0;
  if (live)
    for (int i = 0; i < run; ++i) {
      const unsigned long long u = units_of(first + i);
      units += u;
      mass += mass_of(first + i, u);
    }
  auto up = [&](unsigned long long& v) {
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
  };
  unsigned long long mass_to = mass, units_to = units;
  up(mass_to);
  up(units_to);
  if (lane == 31) {
    sh.sums[warp][0] = mass_to;
    sh.sums[warp][1] = units_to;
  }
  __syncthreads();
  unsigned long long all = 0, all_units = 0, mass_at = *above, units_at = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) {
      mass_at += sh.sums[i][0];
      units_at += sh.sums[i][1];
    }
    all += sh.sums[i][0];
    all_units += sh.sums[i][1];
  }
  turn ^= 1;
  if ((int)threadIdx.x < row.ctas) {
    st_dsmem_u64(dsmem_addr(smem_u32(&sh.box[turn].f64[row.rank][0]), threadIdx.x), all);
    st_dsmem_u64(dsmem_addr(smem_u32(&sh.box[turn].f64[row.rank][1]), threadIdx.x), all_units);
  }
  row.meet();
  unsigned long long everything = *above;
  for (int r = 0; r < row.ctas; ++r) {
    const unsigned long long m = (unsigned long long)__double_as_longlong(sh.box[turn].f64[r][0]);
    everything += m;
    if (r >= row.rank) continue;
    mass_at += m;
    units_at += (unsigned long long)__double_as_longlong(sh.box[turn].f64[r][1]);
  }
  mass_at += mass_to - mass;
  units_at += units_to - units;
  const unsigned long long least = (unsigned long long)((target - margin) * kPart), most = (unsigned long long)((target + margin) * kPart);
  // the bin that reaches `least` first, and the one that passes `most`
  if (live && mass_at <= most && mass_at + mass >= least) {
    for (int i = 0; i < run; ++i) {
      const unsigned long long u = units_of(first + i), m = mass_of(first + i, u);
      if (mass_at < least && mass_at + m >= least)
        for (int r = 0; r < row.ctas; ++r) {
          st_dsmem_u32(dsmem_addr(smem_u32(&sh.bin_above), (uint32_t)r), (uint32_t)(first + i));
          st_dsmem_u64(dsmem_addr(smem_u32(&sh.mass_above), (uint32_t)r), mass_at);
          st_dsmem_u64(dsmem_addr(smem_u32(&sh.units_above), (uint32_t)r), units_at);
        }
      if (mass_at <= most && mass_at + m > most)
        for (int r = 0; r < row.ctas; ++r) {
          st_dsmem_u32(dsmem_addr(smem_u32(&sh.bin_below), (uint32_t)r), (uint32_t)(first + i));
          st_dsmem_u64(dsmem_addr(smem_u32(&sh.units_below), (uint32_t)r), units_at + u);
        }
      mass_at += m;
      units_at += u;
    }
  }
  row.meet();
  // the smallest value of a bin and those above it
  auto value_from = [&](int bin) {                            // 33 parts a round, of which lanes tell
    long long a = *lo, b = *hi;
    if (bin_of(place(low)) <= bin) return a;
    while (b - a > 1) {
      const long long mid = a + max((b - a) * (lane + 1) / 33, 1ll);
      const unsigned in = __ballot_sync(0xffffffffu, mid >= b || bin_of(place(Type<T>::value(mid))) <= bin);
      const int pick = in ? __ffs(in) - 1 : 32;
      const long long below = __shfl_sync(0xffffffffu, mid, max(pick - 1, 0)), to = __shfl_sync(0xffffffffu, mid, min(pick, 31));
      if (pick > 0) a = below;
      if (pick < 32) b = min(b, to);
    }
    return b;
  };
  const int bin_above = sh.bin_above, bin_below = sh.bin_below;
  const long long to = bin_above < 0 ? value_from(kBins - 1) : bin_above > 0 ? value_from(bin_above - 1) : *hi;
  if (bin_below >= 0) *lo = value_from(bin_below);
  *hi = to;
  *above = bin_above < 0 ? everything : sh.mass_above;
  return bin_above < 0 || bin_below < 0 ? INFINITY : (double)(sh.units_below - sh.units_above) * 1.01 / (double)one;
}

// The last token that top-p keeps of those x >= from (`more`: what top-k's ties add to their weights), where it lies among
// no more than kFew that fp32 weights cannot tell apart: those are collected and sorted, and the sum and what lies above
// them taken in fp64.  all, largest: fp32's F(from) and F(top).  False: it does not.
template <typename T>
__device__ __noinline__ bool last_kept(const Row<T> row, int& turn, float from, double more, double top_p, double all,
                                       double largest, float* edge, int* last) {
  const float top = sh.weights.top;
  const double about = top_p * (all + more), margin = 4.0 * kOff * about;
  if (!(largest < about - margin) || !(all > about + margin)) return false;
  long long lo = Type<T>::order(fmaxf(from, sh.weights.end)), hi = Type<T>::order(top);
  // How far a histogram's sums may be off, of themselves: by the units' rounding, the bins' weights (2^-18, exp2f of up to 100)
  // and, as the product's factor and the bins' origin are rounded, by 2^-23 of the largest token's share.
  const int bits = min(__clz(row.passes * kThreads * Type<T>::kLanes - 1) - 1, 20);
  const double loose = 1.1 * about * (__hiloint2double((1023 - bits - 1) << 20, 0) + 0x1p-17 + fabs(sh.weights.share) * 0x1p-23);
  double left = INFINITY;
  unsigned long long above = (unsigned long long)(largest * kPart);
  #pragma unroll 1
  for (int time = 0; time < 3 && left > (double)kFew && hi - lo > 1 && (double)above < (about - loose) * kPart; ++time)
    left = narrow<T>(row, turn, about, loose, &lo, &hi, &above, bits, time == 0);
  #pragma unroll 1
  for (int round = 0; left > (double)kFew; ++round) {
    if (round >= 2 || hi - lo <= 1) {
      const double2 n = measure<T, kCount>(row, turn, make_float2(Type<T>::value(lo), Type<T>::value(hi)));
      if (n.x - n.y <= (double)kFew) break;
      if (hi - lo <= 1 || round >= 16) return false;
    }
    long long at[kCuts];
    #pragma unroll
    for (int i = 0; i < kCuts; ++i) {
      at[i] = min(max(lo + (hi - lo) * (i + 1) / (kCuts + 1), lo + 1), hi - 1);
    }
    const double4 q = measure<T, kMass>(row, turn, make_float4(Type<T>::value(at[0]), Type<T>::value(at[1]),
                                                                   Type<T>::value(at[2]), Type<T>::value(at[3])));
    const double g[kCuts] = {q.x, q.y, q.z, q.w};
    bool moved = false;
    #pragma unroll
    for (int i = 0; i < kCuts; ++i) {
      if (g[i] > about + margin && at[i] > lo) {
        lo = at[i];
        moved = true;
      } else if (g[i] < about - margin && at[i] < hi) {
        hi = at[i];
        moved = true;
      }
    }
    if (!moved && round >= 3) return false;                   // and more than kFew in between
  }
  const float below = Type<T>::value(hi);
  const double2 g = measure<T, kExact>(row, turn, make_float2(from, below));
  const unsigned n = collect<T>(row, 2, Type<T>::value(lo), below);
  if (n == 0 || n > kFew) return false;                       // (neither, by the bounds above)
  if (row.rank == 0) {
    sort(n);
    weigh_few(n);
    run_up(n);
    const double target = (top_p * (g.x + more) - g.y) * kWhole;
    unsigned short_of = 0;
    for (unsigned i = 2 * threadIdx.x; i < 2 * threadIdx.x + 2 && i < n; ++i) short_of += (double)sh.few.upto[i] < target;
    const unsigned pick = cta_count(short_of);
    // exact sums say whether the border lies among these tokens at all, whatever the bounds above are worth
    const bool among = target > 0.0 && pick < n;
    const unsigned long long key = sh.few.key[among ? pick : 0];
    if (threadIdx.x < row.ctas) {
      st_dsmem_u32(dsmem_addr(smem_u32(&sh.edge), threadIdx.x), __float_as_uint(value_of((unsigned)(key >> 32))));
      st_dsmem_u32(dsmem_addr(smem_u32(&sh.index), threadIdx.x), among ? (uint32_t)index_of(key) : 0xFFFFFFFFu);
    }
  }
  row.meet();
  if (sh.index < 0) return false;
  *edge = sh.edge;
  *last = sh.index;
  return true;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Params p, int staged) {
  extern __shared__ uint4 stage[];                            // the part, where it fits
  griddep_launch_dependents();
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  if (ctas > 1) cluster_arrive_relaxed();                     // waited for where the logits have been read
  griddep_wait();
  constexpr int kLanes = Type<T>::kLanes;
  Row<T> row;
  row.ctas = (int)ctas;
  row.rank = (int)cluster_rank();
  int turn = 0;
  const int line = (int)(blockIdx.x / ctas);
  const int runs = (p.vocab + kLanes - 1) / kLanes, mine = (runs + row.ctas - 1) / row.ctas;
  row.first = min(row.rank * mine * kLanes, p.vocab);
  row.count = min(mine * kLanes, p.vocab - row.first);
  row.passes = (mine + kThreads - 1) / kThreads;
  row.src = static_cast<const T*>(p.logits) + (long long)line * p.stride + row.first;
  row.vec = p.vec != 0;
  if (threadIdx.x < 16) roots[threadIdx.x] = kRoots[threadIdx.x];
  if (threadIdx.x < 3) sh.here[threadIdx.x] = sh.count[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.unsure = 0;

  double heat = p.temperature ? (double)p.temperature[line] : p.temperature_all;
  Filters filters;
  filters.top_p = p.top_p ? (double)p.top_p[line] : p.top_p_all;
  filters.top_k = p.top_k ? (long long)p.top_k[line] : p.top_k_all;
  const double min_p = p.min_p ? (double)p.min_p[line] : p.min_p_all;
  const double u = fmin(fmax((double)p.uniform[line], 0.0), 1.0);
  const bool greedy = !(heat > 0.0);
  if (!greedy) heat = fmax(heat, 1e-200);      // its inverse is a number; no two fp32 logits are as near as 700 of it
  const bool k_on = filters.top_k > 0 && filters.top_k < p.vocab, p_on = filters.top_p < 1.0, m_on = min_p > 0.0;
  if (!k_on) filters.top_k = 0;
  if (!p_on) filters.top_p = 1.0;
  long long* id = p.ids + line;
  float* logprob = p.logprobs ? p.logprobs + line : nullptr;
  // what takes fp64's slow operations, by a thread that then waits least
  double below = 0.0;                // min-p: w >= min_p where x >= top + T log(min_p)
  if (threadIdx.x == kThreads - 1 && !greedy) {
    sh.weights.set_heat(heat);
    if (m_on) below = heat * log(fmin(min_p, 1.0));
  }

  // the largest logit; the part into shared memory, each thread its own runs
  float most = -INFINITY;
  {
    constexpr int kAhead = 4;
    #pragma unroll 1
    for (int v = 0; v < row.passes; v += kAhead) {
      uint4 r[kAhead];
      #pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (v + i < row.passes) r[i] = row.load(v + i);
      #pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (v + i < row.passes) {
          if (staged) stage[(v + i) * kThreads + threadIdx.x] = r[i];
          float x[kLanes];
          Type<T>::decode(r[i], x);
          #pragma unroll
          for (int e = 0; e < kLanes; ++e) most = fmaxf(most, x[e]);
        }
    }
  }
  if (staged) {
    row.src = reinterpret_cast<const T*>(stage);
    row.count = row.passes * kThreads * kLanes;               // filled up with minus infinity
    row.vec = true;
  }
  row.mine = most = most + 0.f;
  // the largest, and the least of the threads' largest (of those that have some); the row's other CTAs run by now
  if (ctas > 1) cluster_wait();
  uint32_t ends[2] = {order_of(most), most > -INFINITY ? ~order_of(most) : 0u};
  all_u32<T, 2>(row, turn, ends, 0u, [](uint32_t v) { return __reduce_max_sync(0xffffffffu, v); });
  const float top = value_of(ends[0]), least = value_of(~ends[1]);
  if (!(top > -INFINITY)) {
    if (row.rank == 0 && threadIdx.x == 0) {
      *id = -1;
      if (logprob) *logprob = -INFINITY;
    }
    return;                          // no CTA writes to another's shared memory any more
  }
  if (greedy) {
    unsigned at = 0xFFFFFFFFu;
    row.each_of(row.mine == top, [&](const float (&x)[kLanes], int index) {
      #pragma unroll
      for (int e = 0; e < kLanes; ++e)
        if (x[e] == top) at = min(at, (unsigned)(index + e));
    });
    uint32_t v[1] = {at};
    all_u32<T, 1>(row, turn, v, 0xFFFFFFFFu, [](uint32_t x) { return __reduce_min_sync(0xffffffffu, x); });
    if (row.rank == 0 && threadIdx.x == 0) {
      *id = (long long)v[0];
      if (logprob) *logprob = 0.f;
    }
    return;
  }
  const float floor = top == INFINITY ? top : Type<T>::lowest();
  if (threadIdx.x == kThreads - 1) {
    sh.weights.set_top(top, heat);
    sh.edge = m_on && top < INFINITY ? fmaxf(floor, __double2float_ru((double)top + below)) : floor;
  }
  __syncthreads();
  filters.cut = sh.edge;
  const bool fine = sh.weights.fine();
  double2 f = {};                    // fp32's sums over all tokens, and over the largest
  if (p_on && !k_on && fine) f = measure<T, kMass>(row, turn, make_float2(floor, top));

  // ------------------------------------------------------------- few are kept
  if (k_on || p_on || m_on) {
    float from = floor;
    unsigned n = kFew + 1;
    if (p.vocab <= kFew) {
      n = collect<T>(row, 0, floor, NAN);
    } else if (m_on && !(k_on && p_on)) {
      n = collect<T>(row, 0, filters.cut, NAN);
    }
    if (n > kFew && ((k_on && filters.top_k <= kFew / 2) || (p_on && !k_on && fine))) {
      if (bound<T>(row, turn, !k_on, least, k_on ? (double)filters.top_k : fmax(filters.top_p, 0.0) * f.x * (1.0 + 0x1p-16), &from))
        n = collect<T>(row, 1, from, NAN);
    }
    if (n <= kFew) {
      double sum = f.x, off = p_on && !k_on ? kOff : 0.0;
      if (p_on && !k_on && !fine) {
        sum = measure<T, kExact>(row, turn, make_float2(floor, NAN)).x;
        off = 0.0;
      }
      #pragma unroll 1
      for (int time = 0;; ++time) {
        if (row.rank == 0) {
          if (time == 0 && n <= kFewer) weigh_few(n);
          if (!finish(n, filters, sum, off, u, id, logprob) && threadIdx.x < row.ctas)
            st_dsmem_u32(dsmem_addr(smem_u32(&sh.unsure), threadIdx.x), 1u);
        }
        row.meet();
        if (off == 0.0 || !sh.unsure) return;
        sum = measure<T, kExact>(row, turn, make_float2(floor, NAN)).x;
        off = 0.0;
      }
    }
  }

  // ------------------------------------------------------------ many are kept
  // x > edge, and of the tokens that equal it the first `ties` (infinity: all), up to index `last`
  float edge = floor;
  double ties = INFINITY, above;
  int last = 0x7FFFFFFF;
  if (k_on) {
    const double n = measure<T, kCount>(row, turn, make_float2(floor, NAN)).x;
    if (n > (double)filters.top_k) {
      edge = search<T, kCount>(row, turn, floor, (double)filters.top_k, &above);
      ties = (double)filters.top_k - above;
    }
  }
  if (p_on) {
    // sums over what is kept so far: the tokens above `edge` and its ties, or all from `edge` on
    const bool some = ties < INFINITY;
    const float from = !some ? edge : edge < top ? Type<T>::value(Type<T>::order(edge) + 1) : NAN;     // NaN: nothing
    const double top_p = fmax(filters.top_p, 0.0);
    const double w_edge = sh.weights.wide(edge), more = some ? ties * w_edge : 0.0;
    if (fine && k_on) f = measure<T, kMass>(row, turn, make_float2(from, top));
    if (fine && last_kept<T>(row, turn, from, more, top_p, f.x, f.y, &edge, &last)) {
      ties = INFINITY;
    } else {
      f = measure<T, kExact>(row, turn, make_float2(from, top));
      const double target = top_p * (f.x + more);
      if (f.y >= target) {                               // the last one kept is one of the largest
        edge = top;
        ties = fmax(ceil(target), 1.0);
      } else if (!some || f.x >= target) {
        edge = search<T, kExact>(row, turn, from, target, &above);
        ties = fmax(ceil((target - above) / sh.weights.wide(edge)), 1.0);
      } else {                                           // one of the ties at the edge of top-k
        ties = fmin(ties, fmax(ceil((target - f.x) / w_edge), 1.0));
      }
    }
  }
  if (filters.cut > edge) {
    edge = filters.cut;
    ties = INFINITY;
    last = 0x7FFFFFFF;
  }
  if (ties < INFINITY) {
    const double n = locate<T, kCount>(row, turn, edge, 0, ties - 1.0, [&](int i, float, double) {
      for (int r = 0; r < row.ctas; ++r) st_dsmem_u32(dsmem_addr(smem_u32(&sh.index), (uint32_t)r), (uint32_t)i);
    });
    row.meet();
    if (n > ties) last = sh.index;
  }
  // (weights below 2^-100 count only where the token is among the first 2^-40)
  const bool first = fine && u >= 0x1p-40;
  if (first) draw<T, kMass>(row, turn, edge, last, u, id, logprob);
  if (!first || sh.unsure) draw<T, kExact>(row, turn, edge, last, u, id, logprob);
}

}  // namespace smp
}  // namespace ql
