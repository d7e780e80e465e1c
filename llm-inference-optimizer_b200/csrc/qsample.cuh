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
//                   reaches a target: it is searched for over the type's values in
//                   their order, which are whole numbers, with four thresholds a
//                   round, each round a pass.
//
// A token is drawn, or not, by the comparison of two running sums, so these are
// held to more than fp32.  Sums over many weights are first taken, in fp64, of
// weights in fp32, which says how they compare unless they come closer than
// 2^-18.5 of themselves; then the weights are taken again in fp64.
#pragma once

#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "ql_common.cuh"

namespace ql {
namespace smp {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCtas = 16;         // of a row: the largest cluster
constexpr int kMaxPasses = 192;      // 16-byte loads a thread
constexpr int kCuts = 4;             // thresholds of a round
constexpr int kMine = 16;            // thresholds of a round over the threads' largest logits
constexpr int kFew = 1024;           // tokens that one CTA sorts
constexpr double kOff = 1.35e-6;     // 2^-19.5: what sums of fp32 weights may be off, of themselves

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

// exp((x - top) / T) in fp64; infinity less itself counts as 0.
__device__ __noinline__ double exact_weight(float x, float top, double inv_t) {
  const double a = fmin(((double)x - (double)top) * inv_t, 0.0);
  return a < -700.0 ? 0.0 : exp(a);
}

// log(2)^k / k!: 2^r = sum over k of these times r^k.
__host__ __device__ constexpr double taylor(int k) {
  double c = 1.0;
  for (int i = 1; i <= k; ++i) c *= 0.69314718055994530942 / i;
  return c;
}

struct Shared {
  union {                            // what the cluster's CTAs have sent, in turn
    double f64[2][kMaxCtas][kCuts];
    uint32_t u32[2][kMaxCtas][kMine];
  } box;
  union {
    double f64[kWarps][kCuts];
    uint32_t u32[kWarps][kMine];
  } part;
  union {
    double block[kMaxPasses * kWarps];   // of many tokens: sums by runs of the warps
    struct {                         // of few, in the cluster's first CTA
      unsigned long long key[kFew];
      double weight[kFew], upto[kFew];
    } few;
  };
  double before, scan[kWarps];
  unsigned long long found[kFew];    // tokens that this CTA has collected
  unsigned here[3], at, count[3];    // their number, their place in the first CTA's list; the list's length
  int owner, run, index, unsure;
  float edge;
};

// The CTA's part of a row, PASSES 16-byte runs a thread in registers (0: read
// anew in every pass).  Run v of a thread lies v * kThreads runs behind its first.
template <typename T, int PASSES>
struct Part {
  static constexpr int kLanes = Type<T>::kLanes;
  uint4 raw[PASSES > 0 ? PASSES : 1];
  const T* src;
  int first, count, passes;          // of the row: the part's first token, its tokens; runs a thread
  bool vec;

  __device__ __forceinline__ uint4 load(int v) const {
    const int o = (v * kThreads + (int)threadIdx.x) * kLanes;
    if (vec && o + kLanes <= count) return ldg_cg_v4(src + o);
    uint4 r;
    T* e = reinterpret_cast<T*>(&r);
    #pragma unroll
    for (int i = 0; i < kLanes; ++i) e[i] = o + i < count ? src[o + i] : (T)(-INFINITY);
    return r;
  }
  __device__ __forceinline__ void read() {
    if constexpr (PASSES > 0) {
      #pragma unroll
      for (int v = 0; v < PASSES; ++v) raw[v] = load(v);
    }
  }
  __device__ __forceinline__ uint4 run(int v) const {
    if constexpr (PASSES == 0) return load(v);
    uint4 r = raw[0];
    #pragma unroll
    for (int i = 1; i < PASSES; ++i)
      if (v == i) r = raw[i];
    return r;
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {       // f(run, its values)
    float x[kLanes];
    if constexpr (PASSES > 0) {
      #pragma unroll
      for (int v = 0; v < PASSES; ++v) {
        Type<T>::decode(raw[v], x);
        f(v, x);
      }
    } else {
      // four runs on their way at a time
      constexpr int kAhead = 4;
      int v = 0;
      #pragma unroll 1
      for (; v + kAhead <= passes; v += kAhead) {
        uint4 r[kAhead];
        #pragma unroll
        for (int i = 0; i < kAhead; ++i) r[i] = load(v + i);
        #pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          Type<T>::decode(r[i], x);
          f(v + i, x);
        }
      }
      #pragma unroll 1
      for (; v < passes; ++v) {
        Type<T>::decode(load(v), x);
        f(v, x);
      }
    }
  }
  __device__ __forceinline__ int index(int v) const { return first + (v * kThreads + (int)threadIdx.x) * kLanes; }
};

__device__ __forceinline__ unsigned order_of(float x) { return (unsigned)Type<float>::order(x); }
__device__ __forceinline__ float value_of(unsigned k) { return Type<float>::value(k); }

template <typename T, int PASSES>
struct Sampler {
  static constexpr int kLanes = Type<T>::kLanes;
  Part<T, PASSES> part;
  Shared& sh;
  int rank, ctas, turn;              // turn: of the box's two sides
  float top, mine;                   // the row's largest logit, this thread's
  double inv_t, scale, top_scaled;   // 1 / T, log2(e) / T, and that times top
  float scale_hi, scale_lo, low;     // log2(e) / T in two parts; x - top where fp32 weights end
  float slow;                        // x - top below which fp64 weights take exact_weight
  int collected;

  // ------------------------------------------------------------------ weights
  // In fp32, 2^a with a = (x - top) log2(e) / T: a's nearest whole number n, and 2^(a - n), a - n being exact but for its
  // last bits (two parts of the scale).  Weights end at 2^-100.  How far sums of them may be off, of themselves:
  //   2^-22     each 2^(a - n), by ex2.approx
  //   2^-20.5   x - top's rounding, 2^-24 |a| log(2) of each weight: over a sum that has the largest, 1, and up to 2^21 tokens
  //             more, |a| weighs in with 16.3 at most (all of them at a = -18)
  //   2^-22     four added in fp32, two such sums added
  // together 1.2e-6; kOff is 1.35e-6.
  __device__ __forceinline__ float weight(float x) const {
    const float d = fmaxf(x - top, low);
    const float m = fmaf(d, scale_hi, 12582912.f), n = m - 12582912.f;
    const float rest = fmaf(d, scale_lo, fmaf(d, scale_hi, -n));
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(rest));
    return __int_as_float(__float_as_int(w) + (__float_as_int(m) << 23));
  }
  // In fp64: the same, with the series of 2^r at |r| <= 1/2 up to r^11 (the rest is below 2^-46).  x becomes fp64 by its
  // bits: the conversion's own instruction has a quarter of the rate.  (Numbers below fp32's normal ones, and 0, come out
  // as one of their size: 2^-126 of a logit.)
  __device__ __forceinline__ double weight64(float x) const {
    if (!(x - top >= slow)) return exact_weight(x, top, inv_t);
    const unsigned b = __float_as_uint(x);
    const double wide = __hiloint2double((int)(((b & 0x7FFFFFFFu) >> 3) + (896u << 20) | (b & 0x80000000u)), (int)(b << 29));
    const double a = fma(wide, scale, -top_scaled);
    const double m = a + 6755399441055744.0, r = a - (m - 6755399441055744.0);
    double y = taylor(11);
    #pragma unroll
    for (int k = 10; k >= 0; --k) y = fma(y, r, taylor(k));
    return __hiloint2double(__double2hiint(y) + (__double2loint(m) << 20), __double2loint(y));
  }
  template <bool EXACT>
  __device__ __forceinline__ auto weigh(float x) const {
    if constexpr (EXACT) return weight64(x);
    else return weight(x);
  }

  // ------------------------------------------------- sums over the cluster
  __device__ __forceinline__ void meet() {       // all threads of the cluster
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
  }
  // The same result in all threads.  `op` of a warp's 32 values, the same in all its lanes.
  template <int N, typename Op>
  __device__ __forceinline__ void all_u32(uint32_t (&v)[N], uint32_t none, Op op) {
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
        if (lane < ctas) st_dsmem_u32(dsmem_addr(smem_u32(&sh.box.u32[turn][rank][i]), (uint32_t)lane), s);
      }
    }
    meet();
    #pragma unroll
    for (int i = 0; i < N; ++i) v[i] = op(lane < ctas ? sh.box.u32[turn][lane][i] : none);
  }
  template <int N>
  __device__ __forceinline__ void all_count(uint32_t (&v)[N]) {
    all_u32<N>(v, 0u, [](uint32_t x) { return __reduce_add_sync(0xffffffffu, x); });
  }
  __device__ __forceinline__ static double warp_sum(double v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  template <int N>
  __device__ __forceinline__ void all_sum(double (&v)[N]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = warp_sum(v[i]);
      if (lane == 0) sh.part.f64[warp][i] = v[i];
    }
    __syncthreads();
    turn ^= 1;
    if (warp == 0) {
      #pragma unroll
      for (int i = 0; i < N; ++i) {
        const double s = warp_sum(lane < kWarps ? sh.part.f64[lane][i] : 0.0);
        if (lane < ctas) st_dsmem_f64(dsmem_addr(smem_u32(&sh.box.f64[turn][rank][i]), (uint32_t)lane), s);
      }
    }
    meet();
    #pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < ctas ? sh.box.f64[turn][lane][i] : 0.0);
  }

  // F at each threshold: the number of tokens x >= cut, or the sum of their weights.
  template <bool MASS, bool EXACT, int N>
  __device__ __forceinline__ void measure(const float (&cut)[N], double (&f)[N]) {
    uint32_t n[N] = {};
    #pragma unroll
    for (int i = 0; i < N; ++i) f[i] = 0.0;
    part.each([&](int, const float (&x)[kLanes]) {
      float s[2][N] = {};
      #pragma unroll
      for (int e = 0; e < kLanes; ++e) {
        const auto w = MASS ? weigh<EXACT>(x[e]) : 0.f;
        #pragma unroll
        for (int i = 0; i < N; ++i)
          if (x[e] >= cut[i]) {                            // not of a NaN
            if (!MASS) ++n[i];
            else if (EXACT) f[i] += w;
            else s[e & 1][i] += w;
          }
      }
      if (MASS && !EXACT)
        #pragma unroll
        for (int i = 0; i < N; ++i) f[i] += (double)(s[0][i] + s[1][i]);
    });
    if constexpr (MASS) {
      all_sum<N>(f);
    } else {
      all_count<N>(n);
      #pragma unroll
      for (int i = 0; i < N; ++i) f[i] = (double)n[i];
    }
  }

  // The largest value whose F reaches `target`, from F(from) >= target on; *above: F of what lies above it.
  template <bool MASS>
  __device__ __forceinline__ float search(float from, double target, double* above) {
    long long lo = Type<T>::order(from), hi = Type<T>::order(top) + 1;
    *above = 0.0;
    while (hi - lo > 1) {
      long long at[kCuts];
      float cut[kCuts];
      double f[kCuts];
      #pragma unroll
      for (int i = 0; i < kCuts; ++i) {
        at[i] = lo + max((hi - lo) * (i + 1) / (kCuts + 1), 1ll);
        cut[i] = Type<T>::value(at[i]);
      }
      measure<MASS, MASS>(cut, f);
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
  template <bool MASS>
  __device__ __forceinline__ bool bound(float least, double target, float* v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr float kUnit = 0x1p22f;                          // weights are counted in whole units: never too much
    const uint32_t unit = MASS ? (uint32_t)(weight(mine) * kUnit) : 1u;
    const double wanted = MASS ? target * (double)kUnit : target;
    long long lo = Type<T>::order(least), hi = Type<T>::order(top) + 1;
    bool found = false;
    for (int round = 0; round < 10; ++round) {
      const long long at = lo + (hi - lo) * (lane & (kMine - 1)) / kMine;
      const float cut = Type<T>::value(at);
      uint32_t f = 0;
      #pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const bool over = mine >= __shfl_sync(0xffffffffu, cut, i);
        const uint32_t n = MASS ? __reduce_add_sync(0xffffffffu, over ? unit : 0u) : __popc(__ballot_sync(0xffffffffu, over));
        if (lane == i) f = n;
      }
      if (lane < kMine) sh.part.u32[warp][lane] = f;
      __syncthreads();
      turn ^= 1;
      if (warp == 0 && lane < kMine) {
        f = 0;
        #pragma unroll
        for (int w = 0; w < kWarps; ++w) f += sh.part.u32[w][lane];
        for (int r = 0; r < ctas; ++r) st_dsmem_u32(dsmem_addr(smem_u32(&sh.box.u32[turn][rank][lane]), (uint32_t)r), f);
      }
      meet();
      double all = 0.0;
      for (int r = 0; r < ctas; ++r) all += (double)sh.box.u32[turn][r][lane & (kMine - 1)];
      const unsigned enough = __ballot_sync(0xffffffffu, lane < kMine && all >= wanted);
      if (!found && !(enough & 1u)) return false;
      found = true;                                           // of lo, and so of some threshold
      const int pick = 31 - __clz(enough | 1u);
      const long long next = __shfl_sync(0xffffffffu, at, (pick + 1) & (kMine - 1));
      if (pick + 1 < kMine) hi = next;
      lo = __shfl_sync(0xffffffffu, at, pick);
      all = __shfl_sync(0xffffffffu, all, pick);
      if (hi - lo <= 1 || (MASS ? all <= wanted * 1.02 : all <= wanted * 1.25 + 16.0)) break;
    }
    *v = Type<T>::value(lo);
    return true;
  }

  // ---------------------------------------------------------- many are kept
  // The first token, by index, at which the running sum of weigh(x, index) exceeds target(sum), or the last that has a
  // weight: found(index, x, sum) in one thread of the cluster.  Where a running sum comes closer to the target than sums
  // that are `off` of themselves off can tell, sh.unsure is set in all CTAs, to be read behind the next meeting.
  template <typename Weigh, typename Target, typename Found>
  __device__ __forceinline__ double locate(double off, Weigh weigh, Target target, Found found) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // a block: a run of a warp
    part.each([&](int v, const float (&x)[kLanes]) {
      decltype(weigh(0.f, 0)) s[2] = {};
      #pragma unroll
      for (int e = 0; e < kLanes; ++e) s[e & 1] += weigh(x[e], part.index(v) + e);
      const double all = warp_sum((double)(s[0] + s[1]));
      if (lane == 0) sh.block[v * kWarps + warp] = all;
    });
    __syncthreads();
    turn ^= 1;
    const int blocks = part.passes * kWarps, per_lane = (blocks + 31) / 32;
    double own = 0.0, upto = 0.0;
    if (warp == 0) {
      for (int i = 0; i < per_lane; ++i)
        if (lane * per_lane + i < blocks) own += sh.block[lane * per_lane + i];
      upto = own;
      #pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      const double all = __shfl_sync(0xffffffffu, upto, 31);
      if (lane < ctas) st_dsmem_f64(dsmem_addr(smem_u32(&sh.box.f64[turn][rank][0]), (uint32_t)lane), all);
    }
    meet();
    // each CTA finds whose part holds the token, by the same sums
    double sum = 0.0;
    for (int r = 0; r < ctas; ++r) sum += sh.box.f64[turn][r][0];
    const double t = target(sum);
    if (warp == 0) {
      int owner = -1, last = 0;
      double run = 0.0, before = 0.0, last_before = 0.0;
      for (int r = 0; r < ctas; ++r) {
        const double w = sh.box.f64[turn][r][0];
        if (w > 0.0) {
          last = r;
          last_before = run;
          if (owner < 0 && run + w > t) {
            owner = r;
            before = run;
          }
        }
        run += w;
      }
      if (owner < 0) {
        owner = last;
        before = last_before;
      }
      if (owner == rank) {
        const bool some = own > 0.0;
        const unsigned past = __ballot_sync(0xffffffffu, some && before + upto > t), any = __ballot_sync(0xffffffffu, some);
        if (lane == (past ? __ffs(past) - 1 : 31 - __clz(any))) {
          double run = before + (upto - own), kept = run;
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
      if (lane == 0) sh.owner = owner;
    }
    __syncthreads();
    if (sh.owner == rank && warp == sh.run % kWarps) {
      const int v = sh.run / kWarps;
      const double before = sh.before;
      float x[kLanes];
      double w[kLanes], s = 0.0;
      Type<T>::decode(part.run(v), x);
      #pragma unroll
      for (int e = 0; e < kLanes; ++e) {
        w[e] = (double)weigh(x[e], part.index(v) + e);
        s += w[e];
      }
      double to = s;
      #pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(0xffffffffu, to, o);
        if (lane >= o) to += u;
      }
      const unsigned past = __ballot_sync(0xffffffffu, s > 0.0 && before + to > t), any = __ballot_sync(0xffffffffu, s > 0.0);
      if (lane == (past ? __ffs(past) - 1 : 31 - __clz(any))) {
        double run = before + (to - s), from = run, upto = run;
        float x_pick = x[0];
        int pick = 0;
        bool done = false;
        #pragma unroll
        for (int e = 0; e < kLanes; ++e) {
          if (w[e] > 0.0 && !done) {
            pick = e;
            x_pick = x[e];
            from = run;
            upto = run + w[e];
            done = upto > t;
          }
          run += w[e];
        }
        if (off > 0.0 && (t - from <= 2.0 * off * t || upto - t <= 2.0 * off * t))
          for (int r = 0; r < ctas; ++r) st_dsmem_u32(dsmem_addr(smem_u32(&sh.unsure), (uint32_t)r), 1u);
        found(part.index(v) + pick, x_pick, sum);
      }
    }
    return sum;
  }

  // ----------------------------------------------------------- few are kept
  // The tokens cut <= x < below, as (value, index) in the cluster's first CTA; how many there are (past kFew the list is
  // cut off).  At most three times a row.
  __device__ __forceinline__ unsigned collect(float cut, float below = NAN) {
    const int lane = threadIdx.x & 31;
    unsigned *here = &sh.here[collected], *count = &sh.count[collected];
    ++collected;
    if (__any_sync(0xffffffffu, mine >= cut))
      part.each([&](int v, const float (&x)[kLanes]) {
        unsigned n = 0;
        #pragma unroll
        for (int e = 0; e < kLanes; ++e) n += x[e] >= cut && !(x[e] >= below);
        if (!__any_sync(0xffffffffu, n > 0)) return;
        unsigned to = n;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned u = __shfl_up_sync(0xffffffffu, to, o);
          if (lane >= o) to += u;
        }
        unsigned at = 0;
        if (lane == 31) at = atomicAdd(here, to);
        at = __shfl_sync(0xffffffffu, at, 31) + to - n;
        #pragma unroll
        for (int e = 0; e < kLanes; ++e)
          if (x[e] >= cut && !(x[e] >= below)) {
            if (at < kFew)
              sh.found[at] = (unsigned long long)order_of(x[e] + 0.f) << 32 | (0xFFFFFFFFu - (unsigned)(part.index(v) + e));
            ++at;
          }
      });
    __syncthreads();
    const uint32_t counter = dsmem_addr(smem_u32(count), 0), keys = dsmem_addr(smem_u32(&sh.few.key[0]), 0);
    if (threadIdx.x == 0 && *here > 0) sh.at = atom_dsmem_add(counter, *here);
    __syncthreads();
    for (unsigned i = threadIdx.x; i < *here && sh.at + i < kFew; i += kThreads) st_dsmem_u64(keys + (sh.at + i) * 8u, sh.found[i]);
    meet();
    return ld_dsmem_u32(counter);
  }
  // Sorts key[0 .. n) from the largest down, and weight with it, n <= kFew.  Up to 128 by their ranks, four or eight threads
  // counting the larger ones of each; else by merging (64: 1.3 us, by ranks 0.2).
  __device__ __forceinline__ void sort(unsigned n) {
    const unsigned tid = threadIdx.x;
    auto& key = sh.few.key;
    auto& weight = sh.few.weight;
    __syncthreads();
    if (n <= kThreads / 4) {
      const unsigned shift = n <= kThreads / 8 ? 3 : 2, i = tid >> shift, step = 1u << shift;
      const unsigned long long k = i < n ? key[i] : 0;
      const double w = i < n ? weight[i] : 0.0;
      unsigned larger = 0;
      for (unsigned j = tid & (step - 1); j < n; j += step) larger += key[j] > k;
      #pragma unroll
      for (unsigned o = 1; o < 4; o <<= 1) larger += __shfl_xor_sync(0xffffffffu, larger, o);
      if (shift == 3) larger += __shfl_xor_sync(0xffffffffu, larger, 4);
      __syncthreads();
      if (i < n && (tid & (step - 1)) == 0) {
        key[larger] = k;
        weight[larger] = w;
      }
      __syncthreads();
      return;
    }
    unsigned size = kThreads / 2;
    while (size < n) size *= 2;
    for (unsigned i = n + tid; i < size; i += kThreads) key[i] = 0;
    for (unsigned k = 2; k <= size; k *= 2)
      for (unsigned j = k / 2; j > 0; j /= 2) {
        __syncthreads();
        if (tid < size / 2) {
          const unsigned a = 2 * tid - (tid & (j - 1)), b = a + j;
          const unsigned long long x = key[a], y = key[b];
          if ((x < y) == ((a & k) == 0)) {
            key[a] = y;
            key[b] = x;
            const double w = weight[a];
            weight[a] = weight[b];
            weight[b] = w;
          }
        }
      }
    __syncthreads();
  }
  // Weights of key[0 .. n), and both sorted from the largest down.
  __device__ __forceinline__ void sort_by_value(unsigned n) {
    for (unsigned i = threadIdx.x; i < n; i += kThreads)
      sh.few.weight[i] = weight64(value_of((unsigned)(sh.few.key[i] >> 32)));
    sort(n);
  }
  __device__ __forceinline__ static int index_of(unsigned long long key) { return (int)(0xFFFFFFFFu - (unsigned)key); }
  // Running sums of weight[0 .. n) to upto[0 .. n).
  __device__ __forceinline__ void run_up(unsigned n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned i = 2 * threadIdx.x;
    const double a = i < n ? sh.few.weight[i] : 0.0, b = i + 1 < n ? sh.few.weight[i + 1] : 0.0;
    double s = a + b;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) sh.scan[warp] = s;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < warp; ++w) before += sh.scan[w];
    if (i < n) sh.few.upto[i] = before + (s - b);
    if (i + 1 < n) sh.few.upto[i + 1] = before + s;
    __syncthreads();
  }
  // The sum of a count over the CTA.
  __device__ __forceinline__ unsigned cta_count(unsigned n) {
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.part.u32[threadIdx.x >> 5][0] = n;
    __syncthreads();
    n = 0;
    #pragma unroll
    for (int w = 0; w < kWarps; ++w) n += sh.part.u32[w][0];
    return n;
  }
  // The rest, in the first CTA, of n tokens in order that hold all that are kept (and, where `of_few`, all whose weights the
  // sum of top-p is over).  False: `sum` came too close to the weights before some token to tell whether that is kept.
  __device__ __forceinline__ bool finish(unsigned n, long long top_k, double top_p, float cut, double sum, bool of_few, double off,
                                         double u, long long* id, float* logprob) {
    const unsigned tid = threadIdx.x;
    auto& key = sh.few.key;
    auto& weight = sh.few.weight;
    auto& upto = sh.few.upto;
    const unsigned most = top_k > 0 && top_k < (long long)n ? (unsigned)top_k : n;
    run_up(n);
    if (of_few) sum = upto[most - 1];
    const double target = fmax(top_p, 0.0) * sum;
    bool unsure = false;
    unsigned kept = 0;
    for (unsigned i = 2 * tid; i < 2 * tid + 2 && i < most; ++i) {
      const double before = i > 0 ? upto[i - 1] : 0.0;
      if (i > 0 && top_p < 1.0 && fabs(before - target) <= 2.0 * off * target) unsure = true;
      kept += i == 0 || ((top_p >= 1.0 || before < target) && value_of((unsigned)(key[i] >> 32)) >= cut);
    }
    if (__syncthreads_or(unsure && off > 0.0)) return false;
    kept = cta_count(kept);
    const double total = upto[kept - 1], t = u * total;
    // by index
    for (unsigned i = tid; i < kept; i += kThreads) key[i] = key[i] << 32;
    sort(kept);
    run_up(kept);
    // the first whose running sum passes t, else the last that has a weight
    unsigned before = 0;
    for (unsigned i = 2 * tid; i < 2 * tid + 2 && i < kept; ++i) before += upto[i] <= t;
    unsigned pick = cta_count(before);
    if (tid == 0) {
      if (pick >= kept) pick = kept - 1;
      while (pick > 0 && !(weight[pick] > 0.0)) --pick;
      *id = index_of(key[pick] >> 32);
      if (logprob) *logprob = (float)log(weight[pick] / total);
    }
    return true;
  }

  // The last token that top-p keeps of those x >= from (`more`: what top-k's ties add to their weights), where it lies among
  // no more than kFew that fp32 weights cannot tell apart: those are collected and sorted, and the sum and what lies above
  // them taken in fp64.  f: fp32's F(from) and F(top).  False: it does not.
  __device__ __forceinline__ bool last_kept(float from, double more, double top_p, const double (&f)[2], float* edge, int* last) {
    const double about = top_p * (f[0] + more), margin = 4.0 * kOff * about;
    if (!(f[1] < about - margin) || !(f[0] > about + margin)) return false;
    long long lo = Type<T>::order(from), hi = Type<T>::order(top);
    for (int round = 0;; ++round) {
      if (round >= 3 || hi - lo <= 1) {
        const float cuts[2] = {Type<T>::value(lo), Type<T>::value(hi)};
        double n[2];
        measure<false, false>(cuts, n);
        if (n[0] - n[1] <= (double)kFew) break;
        if (hi - lo <= 1 || round >= 16) return false;
      }
      long long at[kCuts];
      float cut[kCuts];
      double g[kCuts];
      #pragma unroll
      for (int i = 0; i < kCuts; ++i) {
        // first by the tokens' weights, from e^-12 to e^-1.5 of the largest
        const long long there = round == 0 ? Type<T>::order(top - (float)((12.0 - 3.5 * i) / inv_t)) : lo + (hi - lo) * (i + 1) / (kCuts + 1);
        at[i] = min(max(there, lo + 1), hi - 1);
        cut[i] = Type<T>::value(at[i]);
      }
      measure<true, false>(cut, g);
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
      if (!moved && round >= 3) return false;                 // and more than kFew in between
    }
    const float cuts[2] = {from, Type<T>::value(hi)};
    double g[2];
    measure<true, true>(cuts, g);
    const unsigned n = collect(Type<T>::value(lo), cuts[1]);
    if (rank == 0) {
      sort_by_value(n);
      run_up(n);
      const double target = top_p * (g[0] + more);
      unsigned short_of = 0;
      for (unsigned i = 2 * threadIdx.x; i < 2 * threadIdx.x + 2 && i < n; ++i) short_of += g[1] + sh.few.upto[i] < target;
      const unsigned pick = min(cta_count(short_of), n - 1);
      if (threadIdx.x < ctas) {
        st_dsmem_u32(dsmem_addr(smem_u32(&sh.edge), threadIdx.x), __float_as_uint(value_of((unsigned)(sh.few.key[pick] >> 32))));
        st_dsmem_u32(dsmem_addr(smem_u32(&sh.index), threadIdx.x), (uint32_t)index_of(sh.few.key[pick]));
      }
    }
    meet();
    *edge = sh.edge;
    *last = sh.index;
    return true;
  }
};

template <typename T, int PASSES>
__global__ void __launch_bounds__(kThreads, PASSES == 0 ? 2 : 1) sample_kernel(const Params p) {
  __shared__ Shared sh;
  griddep_launch_dependents();
  griddep_wait();
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  Sampler<T, PASSES> s = {{}, sh, (int)cluster_rank(), (int)ctas};
  const int row = (int)(blockIdx.x / ctas);
  constexpr int kLanes = Type<T>::kLanes;
  const int runs = (p.vocab + kLanes - 1) / kLanes, mine = (runs + s.ctas - 1) / s.ctas;
  s.turn = 0;
  s.collected = 0;
  if (threadIdx.x < 3) sh.here[threadIdx.x] = sh.count[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.unsure = 0;
  s.part.first = min(s.rank * mine * kLanes, p.vocab);
  s.part.count = min(mine * kLanes, p.vocab - s.part.first);
  s.part.passes = PASSES > 0 ? PASSES : (mine + kThreads - 1) / kThreads;
  s.part.src = static_cast<const T*>(p.logits) + (long long)row * p.stride + s.part.first;
  s.part.vec = p.vec != 0;
  s.part.read();

  const double heat = p.temperature ? (double)p.temperature[row] : p.temperature_all;
  const double top_p = p.top_p ? (double)p.top_p[row] : p.top_p_all;
  const double min_p = p.min_p ? (double)p.min_p[row] : p.min_p_all;
  const long long top_k = p.top_k ? (long long)p.top_k[row] : p.top_k_all;
  const double u = fmin(fmax((double)p.uniform[row], 0.0), 1.0);
  const bool greedy = !(heat > 0.0);
  const bool k_on = !greedy && top_k > 0 && top_k < p.vocab, p_on = !greedy && top_p < 1.0, m_on = !greedy && min_p > 0.0;
  s.inv_t = greedy ? 1.0 : 1.0 / heat;

  float most = -INFINITY;
  s.part.each([&](int, const float (&x)[kLanes]) {
    #pragma unroll
    for (int e = 0; e < kLanes; ++e) most = fmaxf(most, x[e]);
  });
  s.mine = most = most + 0.f;
  float least;
  {
    // the largest, and the least of the threads' largest (of those that have some)
    uint32_t v[2] = {order_of(most), most > -INFINITY ? ~order_of(most) : 0u};
    s.template all_u32<2>(v, 0u, [](uint32_t x) { return __reduce_max_sync(0xffffffffu, x); });
    s.top = value_of(v[0]);
    least = value_of(~v[1]);
  }
  const float top = s.top;
  long long* id = p.ids + row;
  float* logprob = p.logprobs ? p.logprobs + row : nullptr;
  if (!(top > -INFINITY)) {
    if (s.rank == 0 && threadIdx.x == 0) {
      *id = -1;
      if (logprob) *logprob = -INFINITY;
    }
    return;                          // no CTA writes to another's shared memory any more
  }
  if (greedy) {
    unsigned at = 0xFFFFFFFFu;
    if (s.mine == top)
      s.part.each([&](int v, const float (&x)[kLanes]) {
        #pragma unroll
        for (int e = 0; e < kLanes; ++e)
          if (x[e] == top) at = min(at, (unsigned)(s.part.index(v) + e));
      });
    uint32_t v[1] = {at};
    s.template all_u32<1>(v, 0xFFFFFFFFu, [](uint32_t x) { return __reduce_min_sync(0xffffffffu, x); });
    if (s.rank == 0 && threadIdx.x == 0) {
      *id = (long long)v[0];
      if (logprob) *logprob = 0.f;
    }
    return;
  }

  const double scale = s.scale = s.inv_t * 1.4426950408889634074;
  s.top_scaled = (double)top * scale;
  s.slow = (float)(-680.0 * heat);
  s.scale_hi = (float)scale;
  s.scale_lo = (float)(scale - (double)s.scale_hi);
  s.low = fmaxf(-100.f / s.scale_hi, -3.402823466e38f);
  // fp32 weights want a scale that fp32 can square, and no infinite logit
  const bool fine = scale < 0x1p60 && scale > 0x1p-60 && top < INFINITY;
  const float floor = top == INFINITY ? top : Type<T>::lowest();
  // w >= min_p where x >= top + T log(min_p)
  float cut = floor;
  if (m_on && top < INFINITY) cut = fmaxf(floor, __double2float_ru((double)top + heat * log(fmin(min_p, 1.0))));

  double f[2] = {};                  // fp32's sums over all tokens, and over the largest
  if (p_on && !k_on && fine) {
    const float cuts[2] = {floor, top};
    s.template measure<true, false>(cuts, f);
  }

  // ------------------------------------------------------------- few are kept
  if (k_on || p_on || m_on) {
    float from = floor;
    unsigned n = kFew + 1;
    if (p.vocab <= kFew) {
      n = s.collect(floor);
    } else if (m_on && !(k_on && p_on)) {
      n = s.collect(cut);
    }
    if (n > kFew && k_on && top_k <= kFew / 2) {
      if (s.template bound<false>(least, (double)top_k, &from)) n = s.collect(from);
    } else if (n > kFew && p_on && !k_on && fine) {
      if (s.template bound<true>(least, top_p * f[0] * (1.0 + 0x1p-16), &from)) n = s.collect(from);
    }
    if (n <= kFew) {
      double sum = f[0], off = kOff;
      if (p_on && !k_on && !fine) {
        const float cuts[1] = {floor};
        double all[1];
        s.template measure<true, true>(cuts, all);
        sum = all[0];
        off = 0.0;
      }
      if (!p_on || k_on) off = 0.0;
      if (s.rank == 0) {
        s.sort_by_value(n);
        const bool done = s.finish(n, k_on ? top_k : 0, p_on ? top_p : 1.0, cut, sum, k_on, off, u, id, logprob);
        if (!done && threadIdx.x < s.ctas) st_dsmem_u32(dsmem_addr(smem_u32(&sh.unsure), threadIdx.x), 1u);
      }
      s.meet();
      if (off == 0.0 || !sh.unsure) return;
      const float cuts[1] = {floor};
      double all[1];
      s.template measure<true, true>(cuts, all);
      if (s.rank == 0) s.finish(n, 0, top_p, cut, all[0], false, 0.0, u, id, logprob);
      return;
    }
  }

  // ------------------------------------------------------------ many are kept
  // x > edge, and of the tokens that equal it the first `ties` (infinity: all), up to index `last`
  float edge = floor;
  double ties = INFINITY, above;
  int last = p.vocab;
  if (k_on) {
    const float cuts[1] = {floor};
    double n[1];
    s.template measure<false, false>(cuts, n);
    if (n[0] > (double)top_k) {
      edge = s.template search<false>(floor, (double)top_k, &above);
      ties = (double)top_k - above;
    }
  }
  if (p_on) {
    // sums over what is kept so far: the tokens above `edge` and its ties, or all from `edge` on
    const bool some = ties < INFINITY;
    const float from = !some ? edge : edge < top ? Type<T>::value(Type<T>::order(edge) + 1) : NAN;     // NaN: nothing
    const double w_edge = exact_weight(edge, top, s.inv_t), more = some ? ties * w_edge : 0.0;
    const float cuts[2] = {from, top};
    if (fine && k_on) s.template measure<true, false>(cuts, f);
    if (fine && s.last_kept(from, more, fmax(top_p, 0.0), f, &edge, &last)) {
      ties = INFINITY;
    } else {
      s.template measure<true, true>(cuts, f);
      const double target = fmax(top_p, 0.0) * (f[0] + more);
      if (f[1] >= target) {                              // the last one kept is one of the largest
        edge = top;
        ties = fmax(ceil(target), 1.0);
      } else if (!some || f[0] >= target) {
        edge = s.template search<true>(from, target, &above);
        ties = fmax(ceil((target - above) / exact_weight(edge, top, s.inv_t)), 1.0);
      } else {                                           // one of the ties at the edge of top-k
        ties = fmin(ties, fmax(ceil((target - f[0]) / w_edge), 1.0));
      }
    }
  }
  if (cut > edge) {
    edge = cut;
    ties = INFINITY;
    last = p.vocab;
  }
  if (ties < INFINITY) {
    const double n = s.locate(0.0, [&](float x, int) { return x == edge ? 1.f : 0.f; }, [&](double) { return ties - 1.0; },
                              [&](int i, float, double) {
                                for (int r = 0; r < s.ctas; ++r)
                                  st_dsmem_u32(dsmem_addr(smem_u32(&sh.index), (uint32_t)r), (uint32_t)i);
                              });
    s.meet();
    if (n > ties) last = sh.index;
  }
  auto draw = [&](auto exact) {
    constexpr bool kExact = decltype(exact)::value;
    s.locate(kExact ? 0.0 : kOff,
             [&](float x, int i) { return x > edge || (x == edge && i <= last) ? s.template weigh<kExact>(x) : 0; },
             [&](double sum) { return u * sum; },
             [&](int i, float x, double sum) {
               *id = i;
               if (logprob) *logprob = (float)log(exact_weight(x, top, s.inv_t) / sum);
             });
    s.meet();
  };
  if (fine) draw(std::false_type());
  if (!fine || sh.unsure) draw(std::true_type());
}

}  // namespace smp
}  // namespace ql
