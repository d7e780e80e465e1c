// qattend.cuh — attention of a few new tokens per request (one, a chain, or a
// tree of drafted ones) over the quantised paged cache (sm_100a).
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(s_ij) / sum_j exp(s_ij),   s_ij = scale * q_i . k_j
// over the cached positions j that row i sees.  A request's last q_len cached
// positions are its new tokens; row i sees every position before them and,
// of them, those up to i (no mask) or those whose bit is set in its mask row.
// A row that sees nothing gives zeros and a log-sum of minus infinity.
#pragma once

#include <algorithm>
#include <type_traits>

#include "qcache.cuh"
#include "qwork.h"

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
  kvc::Divisor by_group;
  float scale_log2;              // scale * log2(e): scores in units of log2
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
  const long long most = min((long long)p.table_width << p.cache.page_shift, (long long)kMostKeys);
  r.kv_len = (int)min((long long)max(p.kv_lens[b], 0), most);
  return r;
}
__device__ __forceinline__ bool sees(const Params& p, const Request& r, int i, int j) {
  const int d = j - (r.kv_len - r.q_len);        // which new token position j is
  if (!p.mask) return d <= i;
  if (d < 0) return true;
  return d < 64 * p.mask_words && ((p.mask[(long long)(r.q0 + i) * p.mask_words + (d >> 6)] >> (d & 63)) & 1);
}

// ------------------------------------------------------------ work of a launch
// qwork.h says how it is divided; a tile has ROWS = 8 NT rows here.
constexpr float kLow = -1e30f;             // the maximum of nothing: below every score, and finite
constexpr int kWarps = kUnitKeys / 16;     // a warp takes 16 keys of every unit
constexpr int kThreads = 32 * kWarps;
constexpr int kMinUnits = 2;               // units worth a CTA of their own: 256 keys

template <int MIN_UNITS>
__device__ __forceinline__ int item_units(const Request& r) {
  return units_of(r.kv_len, MIN_UNITS);
}
template <int ROWS, int MIN_UNITS>
__device__ __forceinline__ long long request_units(const Params& p, const Request& r) {
  const unsigned tiles = (unsigned)(r.q_len * p.group + ROWS - 1) / ROWS;
  return (long long)tiles * p.cache.heads * item_units<MIN_UNITS>(r);
}

// Sums the requests' units and finds the request that holds this CTA's first
// unit: *b, the unit at which it begins, and its lengths.  All threads call
// it; up to 32 requests each warp does so by itself.
template <int ROWS, int MIN_UNITS, int THREADS>
__device__ __forceinline__ Work find_work(const Params& p, int* b, long long* base, Request* r) {
  __shared__ long long warp_sum[THREADS / 32];
  __shared__ long long found_base;
  __shared__ int found_b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto warp_scan = [&](long long v) {
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  Work w = {0, 0};
  if (p.batch <= 32) {
    Request mine = {0, 0, 0};
    long long units = 0;
    if (lane < p.batch) {
      mine = request(p, lane);
      units = request_units<ROWS, MIN_UNITS>(p, mine);
    }
    const long long incl = warp_scan(units);
    w.total = __shfl_sync(0xffffffffu, incl, 31);
    w.ctas = (int)min((long long)gridDim.x, w.total / MIN_UNITS);
    if ((int)blockIdx.x >= w.ctas) return w;
    const long long u = w.first_unit(blockIdx.x);
    const int at = __ffs(__ballot_sync(0xffffffffu, u < incl)) - 1;      // some lane: u < total
    *b = at;
    *base = __shfl_sync(0xffffffffu, incl - units, at);
    r->q0 = __shfl_sync(0xffffffffu, mine.q0, at);
    r->q_len = __shfl_sync(0xffffffffu, mine.q_len, at);
    r->kv_len = __shfl_sync(0xffffffffu, mine.kv_len, at);
    return w;
  }
  auto scan = [&](long long v, long long* sum) {      // inclusive over the CTA, and its sum
    v = warp_scan(v);
    __syncthreads();
    if (lane == 31) warp_sum[warp] = v;
    __syncthreads();
    long long before = 0, all = 0;
    #pragma unroll
    for (int x = 0; x < THREADS / 32; ++x) {
      if (x < warp) before += warp_sum[x];
      all += warp_sum[x];
    }
    *sum = all;
    return v + before;
  };
  long long mine = 0, incl = 0, sum;
  for (int i = 0; i < p.batch; i += THREADS) {
    const int at = i + threadIdx.x;
    mine = at < p.batch ? request_units<ROWS, MIN_UNITS>(p, request(p, at)) : 0;
    incl = scan(mine, &sum);
    w.total += sum;
  }
  w.ctas = (int)min((long long)gridDim.x, w.total / MIN_UNITS);
  if ((int)blockIdx.x >= w.ctas) return w;
  const long long u = w.first_unit(blockIdx.x);
  long long before = 0;
  for (int i = 0; i < p.batch; i += THREADS) {
    if (p.batch > THREADS) {                          // else mine, incl and sum are still these
      const int at = i + threadIdx.x;
      mine = at < p.batch ? request_units<ROWS, MIN_UNITS>(p, request(p, at)) : 0;
      incl = scan(mine, &sum);
    }
    const long long from = before + incl - mine;
    if (u >= from && u < from + mine) {
      found_b = i + threadIdx.x;
      found_base = from;
    }
    before += sum;
  }
  __syncthreads();
  *b = found_b;
  *base = found_base;
  *r = request(p, *b);
  return w;
}

// ---------------------------------------------------------------- primitives
// 2^x; subnormal results only where a 16-bit type can show them (bf16).
template <bool SUBNORMAL>
__device__ __forceinline__ float ex2(float x) {
  float y;
  if constexpr (SUBNORMAL)
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  else
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Transpose of an 8x8 matrix of 16-bit elements held two to a lane by rows.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// The codes are exact in both 16-bit types.
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_b2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t b2_sub(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// 16-bit lanes of 4 nibbles (codes + 8) -> nibble i of both lanes, fp16
__device__ __forceinline__ void dec4_h(uint32_t u, uint32_t (&v)[4]) {
  const uint32_t w = u >> 8;
  v[0] = h2_sub(lop3_and_or(u, 0x000F000Fu, kH2Magic), kH2_1032);
  v[1] = h2_fma(lop3_and_or(u, 0x00F000F0u, kH2Magic), kH2_1_16, kH2_m72);
  v[2] = h2_sub(lop3_and_or(w, 0x000F000Fu, kH2Magic), kH2_1032);
  v[3] = h2_fma(lop3_and_or(w, 0x00F000F0u, kH2Magic), kH2_1_16, kH2_m72);
}
// the same in bf16: 0x430n is 128 + n
__device__ __forceinline__ void dec4_b(uint32_t u, uint32_t (&v)[4]) {
  #pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = b2_sub(lop3_and_or(u >> (4 * i), 0x000F000Fu, 0x43004300u), 0x43084308u);
}
// 4 signed bytes -> (0, 1), (2, 3) in bf16.  0x43bb with the byte's sign bit
// cleared is 128 + its low 7 bits; with the low 7 bits cleared it is 128, or
// 256 where the sign bit is set: their difference is the signed byte.
__device__ __forceinline__ void dec8_b(uint32_t u, uint32_t& p01, uint32_t& p23) {
  const uint32_t x = __byte_perm(u, 0x43434343u, 0x4140), y = __byte_perm(u, 0x43434343u, 0x4342);
  p01 = b2_sub(x & 0xFF7FFF7Fu, x & 0xFF80FF80u);
  p23 = b2_sub(y & 0xFF7FFF7Fu, y & 0xFF80FF80u);
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a b (+ d unless this begins the sum)
__device__ __forceinline__ void mma_from(float (&d)[4], bool begin, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if (begin)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    mma_16816(d, a0, a1, a2, a3, b0, b1);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
// 16 bytes from global to shared memory, past L1, in the thread's current group.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_if(bool yes, uint32_t dst, const void* src) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p cp.async.cg.shared.global [%0], [%1], 16;\n\t}" ::"r"(dst),
               "l"(src), "r"((int)yes)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {           // all but the newest LEFT groups have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
template <int WORDS>
__device__ __forceinline__ void load_shared(uint32_t (&w)[WORDS], uint32_t addr) {
  if constexpr (WORDS == 1)
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
  else if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr));
}

// Where 16-byte chunk `chunk` of row `row` (of 16) of a tile lies in shared
// memory.  The lanes of a quarter, half or whole warp that read together take
// either neighbouring rows at one place (keys) or every second row at one
// place (values); the order below puts both on different banks.
template <int ROW_BYTES, int BITS>
__device__ __forceinline__ int tile_offset(int row, int chunk) {
  const int u0 = (row ^ (row >> 2)) & 1, u1 = (row >> 1) & 1;      // distinct over rows 4i.., over 0 2 4 6, over 1 3 5 7
  if constexpr (ROW_BYTES == 32) return (row >> 2) * 128 + u1 * 64 + u0 * 32 + chunk * 16;
  if constexpr (ROW_BYTES == 64) return (row >> 1) * 128 + u0 * 64 + (chunk ^ (u1 << 1)) * 16;
  if constexpr (ROW_BYTES == 128 && BITS == 4) return row * 128 + (chunk ^ (u1 << 2) ^ (u0 << 1)) * 16;
  if constexpr (ROW_BYTES == 128 && BITS == 8) return row * 128 + (chunk ^ (row & 6) ^ ((row & 1) << 2)) * 16;
  const int f = ((row >> 1) & 1) ^ ((row & 4)) ^ ((row & 1) << 2);
  return row * 256 + (chunk ^ f) * 16;
}
// tile_offset of a row and chunk that are `drow` and `dchunk` further on,
// where these change no bit that the lane's own row and chunk have set: as a
// constant to xor to the lane's address (tiles are 128-byte aligned) and one
// to add.
template <int ROW_BYTES, int BITS>
__host__ __device__ constexpr int step_xor(int drow, int dchunk) {
  const int r0 = drow & 1, r1 = (drow >> 1) & 1, r2 = (drow >> 2) & 1;
  int x = (dchunk & 7) * 16;
  if (ROW_BYTES == 32) return x ^ r1 * 64 ^ (r0 ^ r2) * 32;
  if (ROW_BYTES == 64) return x ^ (r0 ^ r2) * 64 ^ r1 * 32;
  if (ROW_BYTES == 128 && BITS == 4) return x ^ r1 * 64 ^ (r0 ^ r2) * 32;
  if (ROW_BYTES == 128) return x ^ r1 * 32 ^ r2 * 64 ^ r0 * 64;
  return x ^ r1 * 16 ^ r2 * 64 ^ r0 * 64;
}
template <int ROW_BYTES, int BITS>
__host__ __device__ constexpr int step_add(int drow, int dchunk) {
  if (ROW_BYTES == 32) return (drow >> 2) * 128;
  if (ROW_BYTES == 64) return (drow >> 1) * 128;
  return drow * ROW_BYTES + (dchunk & 8) * 16;
}

// ------------------------------------------------- the kernel for a few rows
// Bound by reading the cache (one unit of keys and values, 33 KB at 8 bits
// and head_dim 128, serves 8 NT rows).  Each warp copies its own tiles of 16
// keys to shared memory some tiles ahead (16-byte asynchronous copies, no
// barrier beyond the warp), and reads them from there straight into the
// registers that the matrix instructions take them from.
//
// Keys are the M side of both products, rows the N side (m16n8k16):
//   S^T[key, row] = K Q^T: lane (g, t) = (lane / 4, lane % 4) holds keys g and
//     g + 8.  The order of the sum over head_dim is free, so a lane reads 16
//     neighbouring elements of a key from each 64 and Q is laid out alike.
//   O^T[d, row] = V^T P: lane (g, t) holds keys 2t, 2t + 1, 2t + 8, 2t + 9 and
//     an eighth of head_dim; pairs of keys are joined by byte permutes, and
//     the order of d within a tile of 16 is free (it only names the outputs).
// The codes enter as exact fp16 integers.  Key scales multiply the scores
// afterwards; bf16 queries become fp16 by a power of two per row (8 significant
// bits fit, down to 2^-32 of the row's largest element; a bf16 body for rows
// that reach further, as one with a branch or as two, made every bf16 call 1 to
// 5 % slower).  Value scales multiply the weights, which are rounded
// to fp16 once, against a power of two that follows the largest scale seen:
// half the products of a sum of two, for an error against 64 bits of 0.00022 to
// 0.00027 of an fp16 output, 0.0002 of that its own rounding, and none that shows
// in bf16.
// A tile with a weight below fp16's normal range (or a hidden key) takes the
// product in bf16 instead, the weights as a sum of two: 16 bits and fp32's
// range, so that no score far below the largest and no mixture of scales
// costs precision; it needs twice the decoding and products.
//
// The running maximum of a row moves only when a score passes it by 4 (weights
// up to 2^4): one vote per 16 keys stands for the reductions, the rescaling
// and the look for hidden keys and small weights, which become rare.
//
// A key's scale is read by its own lanes; hidden keys are removed by
// selection, never by multiplication, so what unused rows of a page hold
// does not matter.
//
// 64 requests of 3152 to 8192 positions, one token, 32 heads over 8 of 128, 8
// bits: 129 us, 5.9 TB/s, 90 % of a plain copy's rate.  Repeated for seconds,
// that draws the GPU's 1000 W; the SM clock falls from 1965 to about 1700 MHz
// and the time rises to 147.  At 4 bits half the bytes want as many
// instructions (about 400 per warp and tile of 16 keys), which bound it: one
// token over 130001 positions, 28 heads over 4: 31 us, of which the tiles take
// 18, the rest being a CTA's start and the joining of parts.
template <int D, int BITS, int NT>
struct Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kChunks = D / 64;
  static constexpr int kGroups = BITS == 8 ? 1 : kChunks;
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kKeyWords = BITS == 8 ? 4 : 2;                // of a 64-element chunk
  static constexpr int kValWords = BITS == 8 ? D / 32 : D / 64;      // of a lane's eighth of a row
  static constexpr int kTiles = D / 16;
  static constexpr int kCtas = D == 256 ? 1 : NT == 1 ? 2 : 1;       // per SM, by registers
  // partial of an item: per row its maximum, its sum and D outputs
  static constexpr int kPartial = kRows * (D + 2);
  // a warp's ring: 16 rows of keys, of values, and their scales, a stage
  static constexpr int kTileBytes = 16 * kRowBytes, kScaleBytes = 16 * kGroups * 2;
  static constexpr int kStageBytes = (2 * (kTileBytes + kScaleBytes) + 127) / 128 * 128;
  static constexpr int kBudget = (kCtas == 2 ? 108 : 216) * 1024;
  // Stages: as many as keep 64 KB on the way to an SM while one is worked on, no more than fit or than 6.  Deeper
  // rings only lengthen the queues (8 bits and head_dim 128, 3 stages: 130.4 us against 128.6 with 2); at 4 bits and
  // head_dim 64, 2 stages are too few (30.6 against 30.2).
  static constexpr int kAll = kCtas * kWarps * kStageBytes, kFit = kBudget / (kWarps * kStageBytes);
  static constexpr int kWant = std::min(1 + (64 * 1024 + kAll - 1) / kAll, 6);
  static constexpr int kStages = std::min(kFit, kWant);
  static_assert(kStages >= 2 && 4 * kGroups <= 32, "");
  static constexpr size_t kRing = (size_t)kWarps * kStages * kStageBytes;
  // rows of the warps to be joined take the ring's place; their stride puts the rows that a quarter warp writes
  // together on different banks
  static constexpr int kRowStride = D + 4;
  static constexpr size_t kJoined = (size_t)kWarps * kRows * (kRowStride + 2) * sizeof(float);
  static constexpr size_t kSmem = 128 + (kRing > kJoined ? kRing : kJoined);
};

template <typename T, int D, int BITS, int NT>
__global__ void __launch_bounds__(kThreads, (Shape<D, BITS, NT>::kCtas))
    stream_kernel(const Params p, unsigned* counters, float* partials) {
  using S = Shape<D, BITS, NT>;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  griddep_launch_dependents();
  griddep_wait();
  extern __shared__ float smem_raw[];
  float* smem = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u) / 4;
  float* sm_o = smem;                                   // [warp][row][kRowStride]
  float* sm_m = smem + kWarps * S::kRows * S::kRowStride;   // [warp][row]
  float* sm_l = sm_m + kWarps * S::kRows;
  __shared__ int last_one;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const kvc::Pool& kv = p.cache;
  int b;
  long long base;
  Request r;
  const Work work = find_work<S::kRows, kMinUnits, kThreads>(p, &b, &base, &r);
  if ((int)blockIdx.x >= work.ctas) return;
  long long u = work.first_unit(blockIdx.x);
  const long long u_end = work.first_unit(blockIdx.x + 1);

  while (u < u_end) {
    // ------------------------------------------------------ the next segment
    long long mine = request_units<S::kRows, kMinUnits>(p, r);
    while (u >= base + mine) {
      base += mine;
      r = request(p, ++b);
      mine = request_units<S::kRows, kMinUnits>(p, r);
    }
    const int per_item = item_units<kMinUnits>(r);
    const int tiles = (int)((unsigned)(r.q_len * p.group + S::kRows - 1) / S::kRows);
    const long long item = Work::quotient(u - base, per_item);
    const int k_begin = (int)((u - base) - item * per_item);
    const int k_end = (int)min((long long)per_item, k_begin + (u_end - u));
    const int head = (int)Work::quotient(item, tiles), row0 = (int)(item - (long long)head * tiles) * S::kRows;
    const int rows = min(S::kRows, r.q_len * p.group - row0);
    const int context = r.kv_len - r.q_len;             // positions that every row sees

    // --------------------------------------------- this warp's tiles of 16 keys
    // tile i: keys j0(i) .. j0(i) + 15, within one page
    const int j_first = k_begin * kUnitKeys + warp * 16;
    const int j_stop = min(k_end * kUnitKeys, r.kv_len);
    const int n_tiles = j_first < j_stop ? (j_stop - j_first + kUnitKeys - 1) / kUnitKeys : 0;
    const int* pages = p.page_table + b * p.table_stride;
    bool any_bad = false;                               // some page so far lies outside the pool
    auto fetch_page = [&](int i) {                      // of tile i + lane
      return i + lane < n_tiles ? pages[(j_first + (i + lane) * kUnitKeys) >> kv.page_shift] : 0;
    };
    auto check_page = [&](int page) {
      const bool bad = page < 0 || page >= p.num_pages;
      if (__any_sync(0xffffffffu, bad)) {
        any_bad = true;
        if (bad) atomicCAS(p.err, 0u, (unsigned)kDevErrBadIndex);
      }
      return bad ? -1 : page;
    };
    int page_now = fetch_page(0), page_next = fetch_page(32), pages_at = 0;   // of tiles 32 pages_at ..
    // rows g of the queries, on their way while the pages are looked up and the first tiles copied
    kvc::Vec8<T> q_raw[NT][S::kChunks][2];
    #pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + 8 * n + g;
      const bool live = 8 * n + g < rows;
      const int token = live ? p.by_group.of(row) : 0, qh = head * p.group + (live ? row - token * p.group : 0);
      const T* src = static_cast<const T*>(p.q.p) + (long long)(r.q0 + token) * p.q.token_stride + qh * p.q.head_stride;
      #pragma unroll
      for (int c = 0; c < S::kChunks; ++c)
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
          const T* at = src + c * 64 + t * 16 + h * 8;
          if (live && p.q.vec) {
            q_raw[n][c][h] = *reinterpret_cast<const kvc::Vec8<T>*>(at);
          } else {
            #pragma unroll
            for (int i = 0; i < 8; ++i) q_raw[n][c][h].v[i] = live ? at[i] : kvc::from_f<T>(0.f);
          }
        }
    }
    page_now = check_page(page_now);
    page_next = check_page(page_next);

    const uint32_t ring = smem_u32(smem) + warp * S::kStages * S::kStageBytes;
    constexpr int kRowChunks = S::kRowBytes / 16;
    const uint32_t copy_at = tile_offset<S::kRowBytes, BITS>(lane / kRowChunks, lane % kRowChunks);
    const uint32_t key_at = BITS == 8 ? tile_offset<S::kRowBytes, BITS>(g, t)
                                      : tile_offset<S::kRowBytes, BITS>(g, t >> 1) + (t & 1) * 8;
    const uint32_t value_at = S::kTileBytes +
        (BITS == 4 ? tile_offset<S::kRowBytes, BITS>(2 * t, g >> 2) + (g & 3) * 4
         : D == 64 ? tile_offset<S::kRowBytes, BITS>(2 * t, g >> 1) + (g & 1) * 8
                   : tile_offset<S::kRowBytes, BITS>(2 * t, g * (D / 128)));
    auto page_of = [&](int i) { return __shfl_sync(0xffffffffu, (i >> 5) == pages_at ? page_now : page_next, i & 31); };
    // Copies of tile i to the stage at `dst` (of a page outside the pool, any rows: its keys are hidden).  A lane's
    // part of a tile, and of the scales: the first lanes take those of the keys, the next of the values.
    const unsigned char *lane_k = kv.k_codes + lane * 16, *lane_v = kv.v_codes + lane * 16;
    const bool of_values = lane >= 2 * S::kGroups;
    const unsigned short* lane_s = (of_values ? kv.v_scales : kv.k_scales) + (lane - (of_values ? 2 * S::kGroups : 0)) * 8;
    const unsigned scale_page = of_values ? kv.vs_page : kv.ks_page;
    auto copy_tile = [&](int i, uint32_t dst) {
      const unsigned page = (unsigned)max(page_of(i), 0);
      const unsigned at = (head << kv.page_shift) + ((j_first + i * kUnitKeys) & ((1 << kv.page_shift) - 1));
      const unsigned char* k = lane_k + (unsigned long long)page * kv.k_page + (unsigned long long)at * S::kRowBytes;
      const unsigned char* v = lane_v + (unsigned long long)page * kv.v_page + (unsigned long long)at * S::kRowBytes;
      const unsigned short* sc = lane_s + (unsigned long long)page * scale_page + (unsigned long long)at * S::kGroups;
      #pragma unroll
      for (int c = 0; c < kRowChunks / 2; ++c) {
        const uint32_t to = ((dst + copy_at) ^ step_xor<S::kRowBytes, BITS>(c * 32 / kRowChunks, 0)) +
                            step_add<S::kRowBytes, BITS>(c * 32 / kRowChunks, 0);
        copy16(to, k + c * 512);
        copy16(to + S::kTileBytes, v + c * 512);
      }
      copy16_if(lane < 4 * S::kGroups, dst + 2 * S::kTileBytes + lane * 16, sc);
    };
    __syncwarp();
    #pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) {
      if (i < n_tiles) copy_tile(i, ring + i * S::kStageBytes);
      copy_commit();
    }

    // ------------------------------------------------------------- queries
    uint32_t qb[NT][S::kTiles][2];
    float rs[NT][2];                                    // on the scores of rows 2t, 2t + 1
    #pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[S::kChunks][16], down = 1.f, up = 1.f;
      unsigned top = 0;
      #pragma unroll
      for (int c = 0; c < S::kChunks; ++c)
        #pragma unroll
        for (int i = 0; i < 16; ++i) {
          f[c][i] = kvc::to_f(q_raw[n][c][i / 8].v[i % 8]);
          if (kBf16) top = max(top, __float_as_uint(f[c][i]) & 0x7FFFFFFFu);
        }
      if constexpr (kBf16) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the row's largest element to 2^15 .. 2^16: what is 2^-32 of it and more keeps its 8 bits, subnormals too
        const int e = top >= 0x7F800000u ? 0 : max((int)(top >> 23) - 127 - 15, -126);
        down = pow2(-e);
        up = pow2(e);
      }
      #pragma unroll
      for (int c = 0; c < S::kChunks; ++c)
        #pragma unroll
        for (int w = 0; w < 4; ++w)
          #pragma unroll
          for (int x = 0; x < 2; ++x) {
            // 8 bits: steps of 4 neighbours; 4 bits: elements i and i + 4 of 8 share a word
            const int i = BITS == 8 ? 4 * w + 2 * x : 8 * (w >> 1) + 2 * (w & 1) + x;
            const int j = BITS == 8 ? i + 1 : i + 4;
            qb[n][4 * c + w][x] = pack_h2(f[c][i] * down, f[c][j] * down);
          }
      #pragma unroll
      for (int x = 0; x < 2; ++x) rs[n][x] = kBf16 ? __shfl_sync(0xffffffffu, up, (2 * t + x) * 4) : 1.f;
    }

    // ---------------------------------------------------------- running state
    float acc[NT][S::kTiles][4];
    float m[NT][2], l[NT][2];
    float v_ref = 0.f, fac = 1.f;                       // power of two at least every value scale seen; on the weights
    bool open = true;                                   // some row has seen nothing yet
    #pragma unroll
    for (int n = 0; n < NT; ++n) {
      #pragma unroll
      for (int i = 0; i < S::kTiles; ++i)
        #pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][i][e] = 0.f;
      #pragma unroll
      for (int x = 0; x < 2; ++x) {
        m[n][x] = 0.f;
        l[n][x] = 0.f;
      }
    }

    uint32_t here = ring + (S::kStages - 1) * S::kStageBytes;
    #pragma unroll 1
    for (int i = 0; i < n_tiles; ++i) {
      const int j0 = j_first + i * kUnitKeys;
      copy_wait<S::kStages - 2>();
      __syncwarp();
      if ((i >> 5) > pages_at) {
        ++pages_at;
        page_now = page_next;
        page_next = check_page(fetch_page(32 * pages_at + 32));
      }
      const bool hidden = any_bad && page_of(i) < 0;
      // the stage before this one, read to its end by all lanes, takes the next tile
      if (i + S::kStages - 1 < n_tiles) copy_tile(i + S::kStages - 1, here);
      copy_commit();
      here = here == ring + (S::kStages - 1) * S::kStageBytes ? ring : here + S::kStageBytes;
      uint32_t kw[2][S::kChunks][S::kKeyWords];
      float ks[2][S::kGroups];
      #pragma unroll
      for (int x = 0; x < 2; ++x) {
        #pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
          constexpr int kStep = BITS == 8 ? 4 : 2;
          load_shared<S::kKeyWords>(kw[x][c], ((here + key_at) ^ step_xor<S::kRowBytes, BITS>(0, kStep * c)) +
                                                  step_add<S::kRowBytes, BITS>(8 * x, kStep * c));
        }
      }
      auto load_scales = [&](float (&sc)[2][S::kGroups], uint32_t at) {
        #pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t addr = at + (g + 8 * x) * S::kGroups * 2;
          if constexpr (S::kGroups == 1) {
            unsigned short h;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(addr));
            sc[x][0] = kvc::bf16_bits_to_f(h);
          } else {
            uint32_t w[S::kGroups / 2];
            load_shared<S::kGroups / 2>(w, addr);
            #pragma unroll
            for (int q = 0; q < S::kGroups; ++q)
              sc[x][q] = __uint_as_float(q & 1 ? w[q / 2] & 0xFFFF0000u : w[q / 2] << 16);
          }
        }
      };
      load_scales(ks, here + 2 * S::kTileBytes);
      // ---------------------- scores, less the rows' maxima, in units of log2
      float d[NT][4];
      #pragma unroll
      for (int n = 0; n < NT; ++n)
        #pragma unroll
        for (int e = 0; e < 4; ++e) d[n][e] = -m[n][e & 1];
      #pragma unroll
      for (int c = 0; c < S::kChunks; ++c) {
        if (BITS == 8 && c > 0) break;                  // one sum over all chunks
        float part[NT][4];
        #pragma unroll
        for (int cc = c; cc < (BITS == 8 ? S::kChunks : c + 1); ++cc)
          #pragma unroll
          for (int w = 0; w < S::kKeyWords; ++w) {
            if constexpr (BITS == 8) {
              uint32_t a0, a1, a2, a3;
              dec_w8(kw[0][cc][w], a0, a2);
              dec_w8(kw[1][cc][w], a1, a3);
              #pragma unroll
              for (int n = 0; n < NT; ++n)
                mma_from(part[n], cc == c && w == 0, a0, a1, a2, a3, qb[n][4 * cc + w][0], qb[n][4 * cc + w][1]);
            } else {
              uint32_t x[4], y[4];
              dec4_h(kw[0][cc][w], x);
              dec4_h(kw[1][cc][w], y);
              #pragma unroll
              for (int h = 0; h < 2; ++h)
                #pragma unroll
                for (int n = 0; n < NT; ++n)
                  mma_from(part[n], w == 0 && h == 0, x[2 * h], y[2 * h], x[2 * h + 1], y[2 * h + 1],
                           qb[n][4 * cc + 2 * w + h][0], qb[n][4 * cc + 2 * w + h][1]);
            }
          }
        const float k0 = ks[0][c] * p.scale_log2, k1 = ks[1][c] * p.scale_log2;
        #pragma unroll
        for (int n = 0; n < NT; ++n)
          #pragma unroll
          for (int e = 0; e < 4; ++e)
            d[n][e] = fmaf(part[n][e], (e < 2 ? k0 : k1) * rs[n][e & 1], d[n][e]);
      }

      float v_sc[2][S::kGroups];
      load_scales(v_sc, here + 2 * S::kTileBytes + S::kScaleBytes);
      uint32_t vw[4][S::kValWords];
      #pragma unroll
      for (int x = 0; x < 4; ++x) {
        constexpr int kLoads = BITS == 4 ? S::kChunks : D == 64 ? 1 : D / 128;
        constexpr int kWords = S::kValWords / kLoads, kStep = BITS == 4 ? 2 : 1;
        #pragma unroll
        for (int c = 0; c < kLoads; ++c) {
          uint32_t w[kWords];
          load_shared<kWords>(w, ((here + value_at) ^ step_xor<S::kRowBytes, BITS>(x & 1, kStep * c)) +
                                     step_add<S::kRowBytes, BITS>((x & 1) + (x >> 1) * 8, kStep * c));
          #pragma unroll
          for (int q = 0; q < kWords; ++q) vw[x][kWords * c + q] = w[q];
        }
      }

      // One vote finds what the plain course below cannot take: hidden keys, a
      // score past its row's maximum by more than 4, one below it by more than
      // 20, a value scale above the reference or under a 32nd of it.
      const bool some_hidden = hidden || j0 + 15 >= context;
      float v_top = v_sc[0][0], v_low = v_sc[0][0], d_top = d[0][0], d_low = d[0][0];
      #pragma unroll
      for (int x = 0; x < 2; ++x)
        #pragma unroll
        for (int q = 0; q < S::kGroups; ++q) {
          v_top = fmaxf(v_top, v_sc[x][q]);
          v_low = fminf(v_low, v_sc[x][q]);
        }
      #pragma unroll
      for (int n = 0; n < NT; ++n)
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
          d_top = fmaxf(d_top, d[n][e]);
          d_low = fminf(d_low, d[n][e]);
        }
      const bool plain = d_top <= 4.f && d_low >= -20.f && v_top <= v_ref && v_low >= v_ref * 0.03125f;
      const bool rare = some_hidden || open || !__all_sync(0xffffffffu, plain);
      if (rare) {
        open = false;
        if (some_hidden) {
          #pragma unroll
          for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = j0 + g + (e >> 1) * 8, row = 8 * n + 2 * t + (e & 1);
              const bool see = !hidden && j < r.kv_len && row < rows && sees(p, r, p.by_group.of(row0 + row), j);
              if (!see) d[n][e] = -INFINITY;
            }
        }
        const unsigned bits = __float_as_uint(fmaxf(v_top, 0.f));
        const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, some_hidden || bits >= 0x7F800000u ? 0u : bits));
        float adjust = 1.f;
        if (most > v_ref) {
          const int e = max((int)((__float_as_uint(most) + 0x007FFFFFu) >> 23) - 127, -100);   // 2^e >= most
          v_ref = e > 127 ? INFINITY : pow2(e);
          adjust = pow2(11 - e) / fac;
          fac = pow2(11 - e);
        }
        #pragma unroll
        for (int n = 0; n < NT; ++n)
          #pragma unroll
          for (int x = 0; x < 2; ++x) {
            // a row's own lanes alone move it, so that its bits do not depend on the other rows
            const unsigned lanes = 0x11111111u << t;
            float top = fmaxf(d[n][x], d[n][2 + x]);
            #pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const bool fresh = !(__ballot_sync(0xffffffffu, l[n][x] > 0.f) & lanes);   // it has seen nothing yet
            float keep = 1.f;
            if (top > 4.f || (fresh && top > -INFINITY)) {
              // rounded down, so that the row's largest weight is 1 at least; scores of 2^25 and more, which m follows
              // in steps of more than 4, are then held to 4
              const float moved = __fadd_rd(m[n][x], top), by = __fsub_rd(moved, m[n][x]);
              m[n][x] = moved;
              #pragma unroll
              for (int e = x; e < 4; e += 2) {
                const float less = d[n][e] - by;
                d[n][e] = less > 4.f ? 4.f : less;
              }
              keep = fresh ? 1.f : ex2<kBf16>(-by);
            } else if (fresh) {
              open = true;
            }
            #pragma unroll
            for (int q = 0; q < S::kTiles; ++q) {
              acc[n][q][x] *= keep * adjust;
              acc[n][q][2 + x] *= keep * adjust;
            }
            l[n][x] *= keep;
          }
        open = __any_sync(0xffffffffu, open);
      }
      // ------------------------------------------------------------ weights
      float a[S::kGroups][NT][4];
      #pragma unroll
      for (int n = 0; n < NT; ++n)
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w = ex2<kBf16>(d[n][e]);
          l[n][e & 1] += w;
          #pragma unroll
          for (int q = 0; q < S::kGroups; ++q) a[q][n][e] = w * (v_sc[e >> 1][q] * fac);
        }
      bool wide = false;
      if (rare) {
        float least = INFINITY;
        #pragma unroll
        for (int n = 0; n < NT; ++n)
          #pragma unroll
          for (int e = 0; e < 4; ++e)
            #pragma unroll
            for (int q = 0; q < S::kGroups; ++q) least = fminf(least, a[q][n][e]);
        wide = some_hidden || __any_sync(0xffffffffu, least < 0x1p-14f);
      }

      // -------------------------------------------------------------- values
      // products of 16 keys' values, decoded by dec8 / dec4, tile by tile of 16 elements
      auto products = [&](auto dec8, auto dec4, auto tile) {
        if constexpr (BITS == 8) {
          #pragma unroll
          for (int q = 0; q < S::kValWords; ++q)
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t sel = h == 0 ? 0x5140 : 0x7362;
              uint32_t a0, a1, a2, a3;
              dec8(__byte_perm(vw[0][q], vw[1][q], sel), a0, a1);
              dec8(__byte_perm(vw[2][q], vw[3][q], sel), a2, a3);
              tile(2 * q + h, 0, a0, a1, a2, a3);
            }
        } else {
          #pragma unroll
          for (int c = 0; c < S::kChunks; ++c)
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t sel = h == 0 ? 0x5410 : 0x7632;
              uint32_t x[4], y[4];
              dec4(__byte_perm(vw[0][c], vw[1][c], sel), x);
              dec4(__byte_perm(vw[2][c], vw[3][c], sel), y);
              tile(4 * c + 2 * h, c, x[0], x[1], y[0], y[1]);
              tile(4 * c + 2 * h + 1, c, x[2], x[3], y[2], y[3]);
            }
        }
      };
      if (!wide) {
        uint32_t pb[S::kGroups][NT][2];
        #pragma unroll
        for (int q = 0; q < S::kGroups; ++q)
          #pragma unroll
          for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int h = 0; h < 2; ++h) pb[q][n][h] = transpose8(pack_h2(a[q][n][2 * h], a[q][n][2 * h + 1]));
        products([](uint32_t u, uint32_t& x, uint32_t& y) { dec_w8(u, x, y); },
                 [](uint32_t u, uint32_t (&v)[4]) { dec4_h(u, v); },
                 [&](int at, int q, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                   #pragma unroll
                   for (int n = 0; n < NT; ++n) mma_16816(acc[n][at], a0, a1, a2, a3, pb[q][n][0], pb[q][n][1]);
                 });
      } else if (!hidden) {
        uint32_t hi[S::kGroups][NT][2], lo[S::kGroups][NT][2];
        #pragma unroll
        for (int q = 0; q < S::kGroups; ++q)
          #pragma unroll
          for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x = d[n][2 * h] == -INFINITY ? 0.f : a[q][n][2 * h];
              const float y = d[n][2 * h + 1] == -INFINITY ? 0.f : a[q][n][2 * h + 1];
              const uint32_t u = pack_b2(x, y);
              hi[q][n][h] = transpose8(u);
              lo[q][n][h] = transpose8(pack_b2(x - __uint_as_float(u << 16), y - __uint_as_float(u & 0xFFFF0000u)));
            }
        products([](uint32_t u, uint32_t& x, uint32_t& y) { dec8_b(u, x, y); },
                 [](uint32_t u, uint32_t (&v)[4]) { dec4_b(u, v); },
                 [&](int at, int q, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                   #pragma unroll
                   for (int n = 0; n < NT; ++n) {
                     mma_bf16(acc[n][at], a0, a1, a2, a3, hi[q][n][0], hi[q][n][1]);
                     mma_bf16(acc[n][at], a0, a1, a2, a3, lo[q][n][0], lo[q][n][1]);
                   }
                 });
      }
    }
    copy_wait<0>();
    __syncthreads();                                    // the ring gives way to the joined rows

    // -------------------------------------------- join the warps of the CTA
    #pragma unroll
    for (int n = 0; n < NT; ++n)
      #pragma unroll
      for (int x = 0; x < 2; ++x) {
        #pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], o);
        if (l[n][x] == 0.f) m[n][x] = kLow;             // nothing seen
        if (g == 0) {
          sm_m[warp * S::kRows + 8 * n + 2 * t + x] = m[n][x];
          sm_l[warp * S::kRows + 8 * n + 2 * t + x] = l[n][x];
        }
      }
    __syncthreads();
    #pragma unroll
    for (int n = 0; n < NT; ++n)
      #pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = 8 * n + 2 * t + x;
        float top = kLow;
        #pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w * S::kRows + row]);
        // one after the other: their product can be too small for fp32
        const float f = ex2<kBf16>(m[n][x] - top), unit = 1.f / fac;
        float* dst = sm_o + (warp * S::kRows + row) * S::kRowStride + g * 4;
        #pragma unroll
        for (int i = 0; i < S::kTiles; i += 2)
          *reinterpret_cast<float4*>(dst + i * 16) =
              make_float4(acc[n][i][x] * unit * f, acc[n][i][2 + x] * unit * f, acc[n][i + 1][x] * unit * f,
                          acc[n][i + 1][2 + x] * unit * f);
      }
    __syncthreads();

    // a row's maximum, sum and output over the warps, in warp order
    const long long item_begin = base + item * per_item;
    const bool whole = k_begin == 0 && k_end == per_item;
    float* mine_out = partials + (long long)(2 * blockIdx.x + (k_begin == 0)) * S::kPartial;
    // Four neighbouring elements of a row are parked at `at`: those of lane group g = at / 4 % 8 and tiles 2 j,
    // 2 j + 1, j = at / 32, which are elements 4 j.. of its eighth (8 bits), or 4 (j % 2).. of its 8 in 64 j / 2 (4 bits).
    auto finish = [&](int row, int place, const float4& o, float top, float sum) {
      const int pg = (place >> 2) & 7, j = place >> 5;
      const int d = BITS == 8 ? pg * (D / 8) + 4 * j : (j >> 1) * 64 + pg * 8 + 4 * (j & 1);
      const int token = p.by_group.of(row0 + row), qh = head * p.group + (row0 + row) - token * p.group;
      const long long at = (long long)(r.q0 + token) * p.q_heads + qh;
      const float f[4] = {o.x, o.y, o.z, o.w};
      kvc::Vec4<T> v;
      #pragma unroll
      for (int i = 0; i < 4; ++i) v.v[i] = kvc::from_f<T>(sum == 0.f ? 0.f : f[i] / sum);
      *reinterpret_cast<kvc::Vec4<T>*>(static_cast<T*>(p.out) + at * D + d) = v;
      if (p.lse && place == 0) p.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718056f;
    };
    auto park = [&](float* dst, int row, int d, const float4& o, float top, float sum) {
      *reinterpret_cast<float4*>(dst + 2 * S::kRows + row * D + d) = o;
      if (d == 0) {
        dst[row] = top;
        dst[S::kRows + row] = sum;
      }
    };
    for (int e = threadIdx.x * 4; e < rows * D; e += kThreads * 4) {
      const int row = e / D, d = e - row * D;
      float top = kLow, sum = 0.f;
      float4 o = {0.f, 0.f, 0.f, 0.f};
      #pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w * S::kRows + row]);
      #pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        sum += sm_l[w * S::kRows + row] * ex2<kBf16>(sm_m[w * S::kRows + row] - top);
        const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * S::kRows + row) * S::kRowStride + d);
        o.x += v.x;
        o.y += v.y;
        o.z += v.z;
        o.w += v.w;
      }
      if (whole)
        finish(row, d, o, top, sum);
      else
        park(mine_out, row, d, o, top, sum);
    }

    if (!whole) {
      const Join j = join_of(work, item_begin, per_item, (int)blockIdx.x);
      auto part = [&](int q) {                          // the first begins the item: its CTA's second slot
        return partials + (long long)(2 * (j.c_first + q) + (q == 0)) * S::kPartial;
      };
      auto arrive = [&](unsigned* counter, int n) {     // true in the last of n CTAs, which sees the others' parts
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
          last_one = atomic_add_acq_rel_gpu(counter, 1u) == (unsigned)n - 1;
          if (last_one) *counter = 0;
        }
        __syncthreads();
        return last_one != 0;
      };
      auto join = [&](int first, int step, int n, auto out) {
        float* f_m = smem;                              // [part][row], then the factors
        float* f_l = smem + n * S::kRows;
        for (int i = threadIdx.x; i < n * S::kRows; i += kThreads) {
          const int q = i / S::kRows, row = i - q * S::kRows;
          if (row < rows) {
            f_m[i] = __ldcg(part(first + q * step) + row);
            f_l[i] = __ldcg(part(first + q * step) + S::kRows + row);
          }
        }
        __syncthreads();
        for (int e = threadIdx.x * 4; e < rows * D; e += kThreads * 4) {
          const int row = e / D, d = e - row * D;
          float top = kLow, sum = 0.f;
          float4 o = {0.f, 0.f, 0.f, 0.f};
          for (int q = 0; q < n; ++q) top = fmaxf(top, f_m[q * S::kRows + row]);
          #pragma unroll 8
          for (int q = 0; q < n; ++q) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(part(first + q * step) + 2 * S::kRows + row * D + d));
            const float f = ex2<kBf16>(f_m[q * S::kRows + row] - top);
            sum += f_l[q * S::kRows + row] * f;
            o.x += v.x * f;
            o.y += v.y * f;
            o.z += v.z * f;
            o.w += v.w * f;
          }
          out(row, d, o, top, sum);
        }
      };
      bool last = true;
      if (j.grouped()) {
        last = arrive(counters + j.group_counter(), j.group_parts);
        if (last)
          join(j.group * kJoin, 1, j.group_parts, [&](int row, int d, const float4& o, float top, float sum) {
            park(part(j.group * kJoin), row, d, o, top, sum);   // read by this thread alone; the row's m and l are in shared memory
          });
      }
      if (last && arrive(counters + j.item_counter(), j.item_arrivals()))
        join(0, j.groups > 1 ? kJoin : 1, j.item_arrivals(), finish);
    }
    __syncthreads();                                    // before the next segment reuses shared memory
    u += k_end - k_begin;
  }
}

}  // namespace att
}  // namespace ql
