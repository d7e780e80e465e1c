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
// All three filters keep a beginning of the order, so what is kept is known by
// its last token: a value v and how many of the tokens equal to v are kept.
// For top-k and top-p, v is the largest value whose measure F(v) over tokens
// x >= v (their number; the sum of their weights) reaches a target: it is
// searched for over the type's values in their order, which are whole numbers,
// with four thresholds a round.  No sorting, no histogram, no atomics: each
// thread keeps its logits in registers, and a round is a pass over those, a sum
// over the CTA's threads and one over the cluster of CTAs that shares a row.
//
// Weights and sums are in fp64: a token is drawn, or not, by the comparison of
// two running sums, and the sums of fp32 weights (2^-24 each) would decide one
// row of some dozen over a large vocabulary otherwise than the definition does.
#pragma once

#include <cuda_bf16.h>

#include "ql_common.cuh"

namespace ql {
namespace smp {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCtas = 16;         // of a row: the largest cluster
constexpr int kMaxPasses = 64;       // 16-byte loads a thread
constexpr int kCuts = 4;             // thresholds of a round

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

struct Shared {
  double box[2][kMaxCtas][kCuts];    // what the cluster's CTAs have sent, in turn
  double part[kWarps][kCuts];
  double sums[kMaxCtas];
  double block[kMaxPasses * kWarps];
  double before;
  long long index;
  int owner, at;
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
      #pragma unroll 1
      for (int v = 0; v < passes; ++v) {
        Type<T>::decode(load(v), x);
        f(v, x);
      }
    }
  }
  __device__ __forceinline__ int index(int v) const { return first + (v * kThreads + (int)threadIdx.x) * kLanes; }
};

__device__ __forceinline__ double warp_sum(double v) {
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int PASSES>
struct Sampler {
  static constexpr int kLanes = Type<T>::kLanes;
  Part<T, PASSES> part;
  Shared& sh;
  int rank, ctas, turn;              // turn: of the box's two sides
  float top;                         // the row's largest logit
  double inv_t;

  __device__ __forceinline__ double weight(float x) const {
    const double a = fmin(((double)x - (double)top) * inv_t, 0.0);      // infinity less itself: none
    return a < -700.0 ? 0.0 : exp(a);
  }

  // Sums over the cluster's threads, the same in all.  MAX: the largest instead.
  template <int N, bool MAX = false>
  __device__ __forceinline__ void all_sum(double (&v)[N]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto add = [](double a, double b) { return MAX ? fmax(a, b) : a + b; };
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      #pragma unroll
      for (int i = 0; i < N; ++i) v[i] = add(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
    if (lane == 0)
      #pragma unroll
      for (int i = 0; i < N; ++i) sh.part[warp][i] = v[i];
    __syncthreads();
    turn ^= 1;
    if (warp == 0) {
      #pragma unroll
      for (int i = 0; i < N; ++i) {
        double s = sh.part[lane & (kWarps - 1)][i];
        #pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) s = add(s, __shfl_xor_sync(0xffffffffu, s, o));
        if (lane < ctas) st_dsmem_f64(dsmem_addr(smem_u32(&sh.box[turn][rank][i]), (uint32_t)lane), s);
      }
    }
    cluster_sync_all();
    if (warp == 0) {
      #pragma unroll
      for (int i = 0; i < N; ++i) {
        double s = lane < ctas ? sh.box[turn][lane][i] : MAX ? -INFINITY : 0.0;
        #pragma unroll
        for (int o = kMaxCtas / 2; o > 0; o >>= 1) s = add(s, __shfl_xor_sync(0xffffffffu, s, o));
        if (lane == 0) sh.sums[i] = s;
      }
    }
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sh.sums[i];
  }

  // F at each threshold: the number of tokens x >= cut, or the sum of their weights.
  template <bool MASS>
  __device__ __forceinline__ void measure(const float (&cut)[kCuts], double (&f)[kCuts]) {
    int n[kCuts] = {};
    #pragma unroll
    for (int i = 0; i < kCuts; ++i) f[i] = 0.0;
    part.each([&](int, const float (&x)[kLanes]) {
      #pragma unroll
      for (int e = 0; e < kLanes; ++e) {
        const double w = MASS ? weight(x[e]) : 0.0;
        #pragma unroll
        for (int i = 0; i < kCuts; ++i)
          if (x[e] >= cut[i]) {                              // not of a NaN
            if (MASS) f[i] += w;
            else ++n[i];
          }
      }
    });
    if (!MASS)
      #pragma unroll
      for (int i = 0; i < kCuts; ++i) f[i] = n[i];
    all_sum<kCuts>(f);
  }

  // The largest value whose F reaches `target`, from F(low) >= target on, and F of what lies above it.
  template <bool MASS>
  __device__ __forceinline__ float search(float low, double target, double* above) {
    long long lo = Type<T>::order(low), hi = Type<T>::order(top) + 1;
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
      measure<MASS>(cut, f);
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

  // The first token, by index, at which the running sum of weigh(x, index) exceeds target(sum), or the last
  // that has a weight: found(index, weight, sum) in one thread of the cluster.
  template <typename Weigh, typename Target, typename Found>
  __device__ __forceinline__ double locate(Weigh weigh, Target target, Found found) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    part.each([&](int v, const float (&x)[kLanes]) {
      double s = 0.0;
      #pragma unroll
      for (int e = 0; e < kLanes; ++e) s += weigh(x[e], part.index(v) + e);
      s = warp_sum(s);
      if (lane == 0) sh.block[v * kWarps + warp] = s;
    });
    __syncthreads();
    turn ^= 1;
    const int blocks = part.passes * kWarps, per_lane = (blocks + 31) / 32;
    double mine = 0.0, upto = 0.0;
    if (warp == 0) {
      for (int i = 0; i < per_lane; ++i)
        if (lane * per_lane + i < blocks) mine += sh.block[lane * per_lane + i];
      upto = mine;
      #pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      const double all = __shfl_sync(0xffffffffu, upto, 31);
      if (lane < ctas) st_dsmem_f64(dsmem_addr(smem_u32(&sh.box[turn][rank][0]), (uint32_t)lane), all);
    }
    cluster_sync_all();
    // each CTA finds whose part holds the token, by the same sums
    if (warp == 0) {
      double s = 0.0, before = 0.0;
      for (int r = 0; r < ctas; ++r) s += sh.box[turn][r][0];
      const double t = target(s);
      int owner = -1, last = 0;
      double run = 0.0, last_before = 0.0;
      for (int r = 0; r < ctas; ++r) {
        const double w = sh.box[turn][r][0];
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
        // of its blocks (a warp's tokens of one run), the one
        const bool some = mine > 0.0;
        const double from = before + (upto - mine);
        unsigned past = __ballot_sync(0xffffffffu, some && before + upto > t), any = __ballot_sync(0xffffffffu, some);
        const int pick = past ? __ffs(past) - 1 : 31 - __clz(any);
        if (lane == pick) {
          double at_sum = from, kept = from;
          int at = -1;
          for (int i = lane * per_lane; i < min((lane + 1) * per_lane, blocks); ++i) {
            const double w = sh.block[i];
            if (w > 0.0) {
              at = i;
              kept = at_sum;
              if (at_sum + w > t) break;
            }
            at_sum += w;
          }
          sh.at = at;
          sh.before = kept;
          sh.sums[1] = t;
        }
      }
      if (lane == 0) {
        sh.owner = owner;
        sh.sums[0] = s;
      }
    }
    __syncthreads();
    const double sum = sh.sums[0];
    if (sh.owner == rank && warp == sh.at % kWarps) {
      const int v = sh.at / kWarps;
      const double t = sh.sums[1], before = sh.before;
      float x[kLanes];
      double w[kLanes], s = 0.0;
      Type<T>::decode(part.run(v), x);
      #pragma unroll
      for (int e = 0; e < kLanes; ++e) {
        w[e] = weigh(x[e], part.index(v) + e);
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
        double run = before + (to - s);
        int pick = 0;
        double w_pick = 0.0;
        bool done = false;
        #pragma unroll
        for (int e = 0; e < kLanes; ++e) {
          if (w[e] > 0.0 && !done) {
            pick = e;
            w_pick = w[e];
            done = run + w[e] > t;
          }
          run += w[e];
        }
        found(part.index(v) + pick, w_pick, sum);
      }
    }
    return sum;
  }
};

template <typename T, int PASSES>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Params p) {
  __shared__ Shared sh;
  griddep_launch_dependents();
  griddep_wait();
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  Sampler<T, PASSES> s = {{}, sh, (int)cluster_rank(), (int)ctas, 0, 0.f, 0.0};
  const int row = (int)(blockIdx.x / ctas);
  constexpr int kLanes = Type<T>::kLanes;
  const int runs = (p.vocab + kLanes - 1) / kLanes, mine = (runs + s.ctas - 1) / s.ctas;
  s.part.first = min(s.rank * mine * kLanes, p.vocab);
  s.part.count = min(mine * kLanes, p.vocab - s.part.first);
  s.part.passes = PASSES > 0 ? PASSES : (mine + kThreads - 1) / kThreads;
  s.part.src = static_cast<const T*>(p.logits) + (long long)row * p.stride + s.part.first;
  s.part.vec = p.vec != 0;
  s.part.read();

  const double heat = p.temperature ? (double)p.temperature[row] : p.temperature_all;
  double top_p = p.top_p ? (double)p.top_p[row] : p.top_p_all;
  double min_p = p.min_p ? (double)p.min_p[row] : p.min_p_all;
  const long long top_k = p.top_k ? (long long)p.top_k[row] : p.top_k_all;
  const double u = (double)p.uniform[row];
  const bool greedy = !(heat > 0.0);
  s.inv_t = greedy ? 1.0 : 1.0 / heat;

  float top = -INFINITY;
  s.part.each([&](int, const float (&x)[kLanes]) {
    #pragma unroll
    for (int e = 0; e < kLanes; ++e) top = fmaxf(top, x[e]);
  });
  double most[1] = {(double)top};
  s.template all_sum<1, true>(most);
  s.top = top = (float)most[0] + 0.f;
  long long id = -1;
  const bool empty = !(top > -INFINITY);
  if (empty) {
    if (s.rank == 0 && threadIdx.x == 0) {
      p.ids[row] = -1;
      if (p.logprobs) p.logprobs[row] = -INFINITY;
    }
  } else {
    // what is kept: x > edge, and the first `ties` tokens that equal it (all: infinity)
    float edge = top == INFINITY ? top : Type<T>::lowest();
    double ties = INFINITY;
    if (greedy) {
      edge = top;
      ties = 1.0;
    } else {
      if (top_k > 0 && top_k < p.vocab) {
        const float cut[kCuts] = {edge, top, top, top};
        double n[kCuts];
        s.template measure<false>(cut, n);
        if (n[0] > (double)top_k) {
          double above;
          edge = s.template search<false>(edge, (double)top_k, &above);
          ties = (double)top_k - above;
        }
      }
      if (top_p < 1.0) {
        // sums over what is kept so far: the tokens above `edge` and its ties, or all from `edge` on
        const bool some = ties < INFINITY;
        const float from = !some ? edge : edge < top ? Type<T>::value(Type<T>::order(edge) + 1) : NAN;   // NaN: nothing
        const float cut[kCuts] = {from, top, NAN, NAN};
        double f[kCuts], above;
        s.template measure<true>(cut, f);
        const double w_edge = s.weight(edge), target = fmax(top_p, 0.0) * (f[0] + (some ? ties * w_edge : 0.0));
        if (f[1] >= target) {                            // the last one kept is one of the largest
          edge = top;
          ties = fmax(ceil(target), 1.0);
        } else if (!some || f[0] >= target) {
          edge = s.template search<true>(from, target, &above);
          ties = fmax(ceil((target - above) / s.weight(edge)), 1.0);
        } else {                                         // one of the ties at the edge of top-k
          ties = fmin(ties, fmax(ceil((target - f[0]) / w_edge), 1.0));
        }
      }
      if (min_p > 0.0) {
        // w >= m where x >= max + T log m
        const double low = (double)top + heat * log(fmin(min_p, 1.0));
        float cut = __double2float_ru(low);
        if (top == INFINITY) cut = top;
        if (cut > edge) {
          edge = cut;
          ties = INFINITY;
        }
      }
    }
    // the index of the last tie kept
    long long last = p.vocab;
    if (ties < INFINITY) {
      const double n = s.locate([&](float x, int i) { return x == edge ? 1.0 : 0.0; }, [&](double) { return ties - 1.0; },
                                [&](int i, double, double) {
                                  for (int r = 0; r < s.ctas; ++r) {
                                    const uint32_t to = dsmem_addr(smem_u32(&sh.index), (uint32_t)r);
                                    asm volatile("st.shared::cluster.s64 [%0], %1;" ::"r"(to), "l"((long long)i) : "memory");
                                  }
                                });
      cluster_sync_all();
      if (n > ties) last = sh.index;
    }
    if (greedy) {
      id = sh.index;
      if (s.rank == 0 && threadIdx.x == 0) {
        p.ids[row] = id;
        if (p.logprobs) p.logprobs[row] = 0.f;
      }
    } else {
      s.locate([&](float x, int i) { return x > edge || (x == edge && i <= last) ? s.weight(x) : 0.0; },
               [&](double sum) { return fmin(fmax(u, 0.0), 1.0) * sum; },
               [&](int i, double w, double sum) {
                 p.ids[row] = i;
                 if (p.logprobs) p.logprobs[row] = (float)log(w / sum);
               });
    }
  }
  cluster_sync_all();                // no CTA leaves while another may write to its shared memory
}

}  // namespace smp
}  // namespace ql
