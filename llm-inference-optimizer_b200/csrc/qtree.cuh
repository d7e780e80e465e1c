// qtree.cuh — attention of many new tokens per request (trees and chains of
// drafted tokens) over the quantised paged cache, on the 5th-generation
// tensor cores (tcgen05 / TMEM, sm_100a).  The mathematics and the division
// of work are those of qattend.cuh; here an item has 256 rows.
//
// With t new tokens under g query heads per key/value head, a key serves t g
// rows: at a few dozen rows the products, not the cache, set the time, and
// mma.sync with one decode per 16 rows is an order of magnitude from the
// tensor cores' rate.  So the codes are decoded once per 256 rows into shared
// memory, as the B operands of
//   S_w [128 rows, keys] = Q_w K^T        (Q_w and K in shared memory)
//   O_w [128 rows, d]   += P_w V          (P_w in TMEM, V in shared memory)
// for two tiles w of 128 rows, and the work is spread over warps:
//   * 4 decode warps: read codes, a step ahead, into registers; decode them
//     exactly to 16 bits and store them in the 128-byte-swizzled layout that
//     both products read (K with d, V with the keys as the sum's direction);
//     publish the step's scales.
//   * 1 warp issues the products: S_0, S_1 of a step, then P_0 V and S_0 of
//     the next, P_1 V and S_1 of the next, so that one tile's softmax runs
//     under the other's products.
//   * 8 softmax warps, a thread a row: S from TMEM, the weights back to TMEM
//     in its place, in two halves, the first multiplied while the second is
//     made.  Key scales multiply the scores, value scales the weights.
// At 4 bits and head_dim 128, where a scale covers 64 elements, a step is 64
// keys with a sum and a set of weights per group.
//
// fp16 calls multiply in fp16, the weights rounded once, which is half the
// products of a sum of two (an output's error against 64 bits is 0.00029 of it,
// 0.00021 of that its own rounding); bf16 calls in bf16, the weights as a sum of
// two (16 bits, fp32's range).  Every wait is bounded;
// after one runs out the others end at once, the loops run to their end
// without meaning, and the device error word tells.
//
// 16 trees of 64 tokens after up to 8133 positions, 28 heads over 4 of 128, 8
// bits, fp16: 139 us, 467 TFLOP/s (bf16: 216 us), 28 % of the tensor cores' rate.  A step
// of 128 keys takes some 4900 cycles, of which its products alone would be
// 2048: P V reads its weights and scores leave through the same TMEM, decode
// and products share the shared memory's ports, and the halves of the softmax
// wait for one another.  About 12 us go into a CTA's start, queries and join (30 while each of a thread's 16 loads of
// queries waited for the one before).
#pragma once

#include "qattend.cuh"
#include "qgemm.cuh"

namespace ql {
namespace tree {

using att::Params;
using att::Request;
using att::Work;

constexpr int kTileRows = 128;
constexpr int kRows = 2 * kTileRows;
constexpr int kMinUnits = 4;             // of 128 keys: a part's outputs are worth 512 keys
constexpr int kSoftmaxWarps = 8, kDecodeWarps = 4, kMmaWarp = kSoftmaxWarps + kDecodeWarps;
constexpr int kThreads = 512;            // the last three warps idle: warpgroups trade registers as a whole

template <int D, int BITS>
struct Shape {
  static constexpr int kAtoms = D / 64;                             // of 64 elements
  static constexpr int kGroups = BITS == 8 ? 1 : kAtoms;
  static constexpr int kKeys = 128 / kGroups;                       // of a step
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kStages = 2 * kGroups;
  static constexpr int kSlots = kStages + 2;                        // of scales: outlive their step's keys
  static constexpr int kQBytes = 2 * kAtoms * kTileRows * 128;
  static constexpr int kStepBytes = kAtoms * kKeys * 128;           // keys, or values, of a step
  static constexpr int kPieces = kKeys * kRowBytes / 16 / (32 * kDecodeWarps);   // 16-byte runs of codes a thread
  static constexpr int kPerPiece = 128 / BITS;                      // elements
  static constexpr int kColumns = 256 + 2 * D;                      // S_0, S_1, O_0, O_1
  // Registers a thread, of the 128 that the launch gives each of 16 warps (8 softmax, 4 decode, 4 with the products'):
  // a softmax thread of one group holds 64 scores, one of two groups 32.
  static constexpr int kSoftmaxRegisters = kGroups > 1 ? 160 : 176, kDecodeRegisters = kGroups > 1 ? 112 : 96,
                       kMmaRegisters = kGroups > 1 ? 80 : 64;
  static_assert(8 * kSoftmaxRegisters + 4 * kDecodeRegisters + 4 * kMmaRegisters <= 16 * 128, "");
  // partial of an item: per row its reference and sum, then D outputs
  static constexpr int kPartial = kRows * (D + 2);
  struct Slot {
    float k[128], v[128];                                           // [group][key]
    float v_log[kKeys];                                             // log2 of a key's largest value scale (kLeast .. kMost)
    unsigned v_top[4];                                              // largest finite value scales
    unsigned bad;                                                   // bit i: keys 16 i .. are in no page
    unsigned pad[3];
  };
  static constexpr size_t kSmem = 1024 + kQBytes + 2 * (size_t)kStages * kStepBytes + kSlots * sizeof(Slot) + 512;
  static_assert(kKeys % 64 == 0 && kPieces >= 1 && kPieces * kPerPiece * 32 * kDecodeWarps == kKeys * D, "");
};

// Where log2 of a value scale ends, so that fp32 follows a row from one end to
// the other.  No fp16 output shows what is below; above, the products have
// room in bf16 (2^(kAim + 61) at most, and sums of 2^21 times 127 of them).
constexpr float kLeast = -32.f, kMost = 60.f;
// log2 of the weight times scale that a row's reference is put at, and of the most that it may come to.
constexpr float kAim = 6.f, kCap = 15.f;

// The products and their commits, by one elected lane of a whole warp in
// uniform control flow: the operands then stay in uniform registers, where a
// branch to one lane would move each of them there anew (140 cycles a product
// under load against 64 of the product itself).
// D[tmem] (+)= A[smem] B[smem], kind::f16.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem].
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrival on `bar` once the products issued so far are done.
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
// Instruction descriptor: fp32 sums, M = 128, N; A and B fp16 or bf16; B's
// rows along the sum (K-major) or along N.
__device__ __forceinline__ uint32_t instruction(bool bf16, bool b_along_n, int n) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_along_n ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTileRows >> 4) << 24);
}
// Shared-memory descriptor of values [key][64 elements] (128-byte rows,
// swizzled): runs of 64 elements lie `atom_bytes` apart, groups of 8 keys 1024.
__device__ __forceinline__ uint64_t desc_values(uint32_t addr, uint32_t atom_bytes) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(atom_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
// Waits for this thread's TMEM loads; the values pass through, so that nothing uses them before.
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
  asm volatile("" : "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                    "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                    "+r"(v[30]), "+r"(v[31]));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// Which of 32 positions from j on row i of the request sees, as bits.
template <bool SHARED>
__device__ __forceinline__ unsigned sees32(const Params& p, const Request& r, int i, int j) {
  const int d0 = j - att::context_of<SHARED>(p, r), left = r.kv_len - j;        // which new token j is; positions left
  const auto low = [](int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; };
  if (!p.mask) return low(min(left, i - d0 + 1));
  unsigned see = 0xFFFFFFFFu;
  if (d0 > -32) {
    const unsigned long long* words = p.mask + (long long)(r.q0 + i) * p.mask_words;
    const auto word = [&](int w) { return w < p.mask_words ? words[w] : 0ull; };
    if (d0 < 0) {
      see = low(-d0) | (unsigned)(word(0) << -d0);
    } else {
      const int sh = d0 & 63;
      see = (unsigned)(word(d0 >> 6) >> sh);
      if (sh > 32) see |= (unsigned)(word((d0 >> 6) + 1) << (64 - sh));
    }
  }
  return see & low(left);
}

template <typename T, int D, int BITS, bool SHARED = false>
__global__ void __launch_bounds__(kThreads, 1) tree_kernel(const Params p, unsigned* counters, float* partials) {
  using S = Shape<D, BITS>;
  using Slot = typename S::Slot;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  constexpr int kTerms = kBf16 ? 2 : 1;
  griddep_launch_dependents();
  griddep_wait();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sm_q = smem;
  uint8_t* sm_k = sm_q + S::kQBytes;
  uint8_t* sm_v = sm_k + S::kStages * S::kStepBytes;
  Slot* slots = reinterpret_cast<Slot*>(sm_v + S::kStages * S::kStepBytes);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(slots + S::kSlots);
  uint64_t* k_free = k_full + S::kStages;
  uint64_t* v_full = k_free + S::kStages;
  uint64_t* v_free = v_full + S::kStages;
  uint64_t* s_full = v_free + S::kStages;                    // per tile
  uint64_t* p_ready = s_full + 2;                            // per tile and half of a step
  uint64_t* half_done = p_ready + 4;                         // the products of a step's first weights
  uint64_t* q_ready = half_done + 2;
  uint64_t* o_done = q_ready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* last_one = reinterpret_cast<int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int b;
  long long base;
  Request r;
  const Work work = att::find_work<kRows, kMinUnits, kThreads, SHARED>(p, &b, &base, &r);
  if constexpr (SHARED) att::clear_early<kThreads>(p);
  if ((int)blockIdx.x >= work.ctas) return;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(k_full + s, kDecodeWarps);
      mbar_init(k_free + s, 1);
      mbar_init(v_full + s, kDecodeWarps);
      mbar_init(v_free + s, 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(s_full + w, 1);
      mbar_init(p_ready + 2 * w, 4);
      mbar_init(p_ready + 2 * w + 1, 4);
      mbar_init(half_done + w, 1);
    }
    mbar_init(q_ready, kSoftmaxWarps);
    mbar_init(o_done, 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) gemm::tmem_alloc(smem_u32(tmem_slot), 512);
  gemm::tc_fence_before();
  __syncthreads();
  gemm::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  static_assert(S::kColumns <= 512, "");

  auto wait = [&](uint64_t* bar, uint32_t parity, unsigned code) {
    if (!mbar_wait(bar, parity & 1, p.err, code, abort)) *abort = 1;
  };

  // Every role goes through the same segments: runs of steps of one item.
  long long u = work.first_unit(blockIdx.x);
  const long long u_end = work.first_unit(blockIdx.x + 1);
  struct Segment {
    long long item_begin;                                    // the item's first unit
    int per_item, k_begin, k_end;                            // its units, and those of the segment
    int head, row0, rows, j_begin, steps;
    bool pair;                                               // more than one tile of rows
  };
  int step = 0, segment = 0;                                 // over the whole launch
  int tile_steps = 0;                                        // a softmax tile's: those in which it took part
  int pair_steps = 0;                                        // the products': those with a second tile
  auto next_segment = [&] {
    Segment g;
    long long mine = att::request_units<kRows, kMinUnits>(p, r);
    while (u >= base + mine) {
      base += mine;
      r = att::request<SHARED>(p, ++b);
      mine = att::request_units<kRows, kMinUnits>(p, r);
    }
    g.per_item = att::item_units<kMinUnits>(r);
    const int tiles = (r.q_len * p.group + kRows - 1) / kRows;
    const long long item = Work::quotient(u - base, g.per_item);
    g.item_begin = base + item * g.per_item;
    g.k_begin = (int)(u - g.item_begin);
    g.k_end = (int)min((long long)g.per_item, g.k_begin + (u_end - u));
    g.head = (int)Work::quotient(item, tiles);
    g.row0 = (int)(item - (long long)g.head * tiles) * kRows;
    g.rows = min(kRows, r.q_len * p.group - g.row0);
    g.j_begin = g.k_begin * att::kUnitKeys;
    const int j_end = min(g.k_end * att::kUnitKeys, r.kv_len);
    g.steps = g.j_begin < j_end ? (j_end - g.j_begin + S::kKeys - 1) / S::kKeys : 0;
    g.pair = g.rows > kTileRows;
    return g;
  };
  auto end_segment = [&](const Segment& g) {
    step += g.steps;
    u += g.k_end - g.k_begin;
    ++segment;
  };

  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kMmaRegisters));
    // what the products' operands depend on, as values that the compiler knows to be the whole warp's
    auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const uint32_t tmem_u = (uint32_t)uniform((int)tmem);
    int done = 0;                                            // steps before the segment
    while (warp == kMmaWarp && uniform(u < u_end)) {
      // ----------------------------------------------------------- products
      const Segment g = next_segment();
      const int steps = uniform(g.steps);
      const bool pair = uniform(g.pair) != 0;
      wait(q_ready, segment, kDevErrMmaWait);
      gemm::tc_fence_after();
      if (steps > 0) {
        const uint32_t q_at = smem_u32(sm_q), k_at = smem_u32(sm_k), v_at = smem_u32(sm_v);
        const uint32_t scores = instruction(kBf16, false, S::kKeys);
        const uint32_t outputs = instruction(kBf16, true, D / S::kGroups);
        auto score = [&](int w, int n) {                     // S_w of step n
          uint64_t qd = gemm::desc_sw128(q_at + (uint32_t)(w * S::kAtoms * kTileRows * 128));
          uint64_t kd = gemm::desc_sw128(k_at + (uint32_t)(n % S::kStages) * S::kStepBytes);
          uint32_t d = tmem_u + (uint32_t)(w * 128);
          #pragma unroll 1
          for (int a = 0; a < S::kAtoms; ++a) {
            #pragma unroll
            for (int i = 0; i < 4; ++i)                      // 32 bytes, 16 elements, along the swizzled rows
              mma_ss(d, qd + 2 * i, kd + 2 * i, scores, i > 0 || (S::kGroups == 1 && a > 0) ? 1u : 0u);
            qd += kTileRows * 128 / 16;
            kd += S::kKeys * 128 / 16;
            if (S::kGroups > 1) d += S::kKeys;
          }
          commit(s_full + w);
        };
        auto output = [&](int w, int n, int half, bool begin) {   // O_w += P_w V over half the keys of step n
          uint64_t vd = desc_values(v_at + (uint32_t)(n % S::kStages) * S::kStepBytes, S::kKeys * 128);
          vd += (uint64_t)(half * S::kKeys * 64 / 16);
          #pragma unroll 1
          for (int q = 0; q < S::kGroups; ++q) {
            uint32_t a = tmem_u + (uint32_t)(w * 128 + q * S::kKeys + half * S::kKeys / 2);
            uint64_t v = vd + (uint64_t)(q * S::kKeys * 128 / 16);
            #pragma unroll 1
            for (int i = 0; i < S::kKeys / 64; ++i) {        // 32 keys: 16 columns of weights and, with two terms, 16 more
              #pragma unroll
              for (int h = 0; h < 2; ++h)
                #pragma unroll
                for (int e = 0; e < kTerms; ++e)
                  mma_ts(tmem_u + (uint32_t)(256 + w * D + q * 64), a + (uint32_t)(h * 8 + e * 16),
                         v + (uint64_t)(h * 2048 / 16), outputs, begin && i == 0 && h == 0 && e == 0 ? 0u : 1u);
              a += 32;
              v += 2 * 2048 / 16;
            }
          }
        };
        // A tile's turn: its weights come in two halves.  The second tile begins when the first has half of its
        // first weights, so that the two stay half a step apart and neither waits for the other's products.
        auto turn = [&](int w, int i, int uses) {
          const int n = done + i, next = n + 1;
          wait(p_ready + 2 * w, uses, kDevErrMmaWait);
          if (w == 0) wait(v_full + n % S::kStages, n / S::kStages, kDevErrMmaWait);
          gemm::tc_fence_after();
          output(w, n, 0, i == 0);
          commit(half_done + w);
          if (w == 0 && i == 0 && pair) score(1, done);
          if (i == 0 && w == (pair ? 1 : 0)) commit(k_free + done % S::kStages);
          wait(p_ready + 2 * w + 1, uses, kDevErrMmaWait);
          gemm::tc_fence_after();
          output(w, n, 1, false);
          if (w == (pair ? 1 : 0)) commit(v_free + n % S::kStages);
          if (i + 1 < steps) {
            if (w == 0) {
              wait(k_full + next % S::kStages, next / S::kStages, kDevErrMmaWait);
              gemm::tc_fence_after();
            }
            score(w, next);
            if (w == (pair ? 1 : 0)) commit(k_free + next % S::kStages);
          }
        };
        wait(k_full + done % S::kStages, done / S::kStages, kDevErrMmaWait);
        gemm::tc_fence_after();
        score(0, done);
        for (int i = 0; i < steps; ++i) {
          turn(0, i, done + i);
          if (pair) turn(1, i, pair_steps + i);
        }
      }
      commit(o_done);
      // nothing of the products is in flight beyond this point, so TMEM can be let go
      wait(o_done, segment, kDevErrMmaWait);
      if (pair) pair_steps += steps;
      done += steps;
      end_segment(g);
    }
  } else if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kDecodeRegisters));
    while (u < u_end) {
      // -------------------------------------------------------------- decode
      const Segment g = next_segment();
      const int steps = g.steps, head = g.head, j_begin = g.j_begin;
      const kvc::Pool& kv = p.cache;
      const int t = threadIdx.x - 32 * kSoftmaxWarps;
      constexpr int kRowPieces = S::kRowBytes / 16, kRowStep = 32 * kDecodeWarps / kRowPieces;
      const int row = t / kRowPieces, piece = t % kRowPieces;          // of pieces row + i kRowStep
      const int* pages = p.page_table + b * p.table_stride;
      const int in_page = (1 << kv.page_shift) - 1;
      // Lane x looks up the page of keys 16 x .. of a step (one of a page outside the pool becomes 0 and a bit of
      // `bad`); a piece's page then comes from the lane of its block.
      constexpr int kBlocks = S::kKeys / 16;
      int page = 0;
      unsigned bad = 0, bad_next = 0;
      auto fetch_pages = [&](int j0) {
        const int j = j0 + (lane & (kBlocks - 1)) * 16;
        page = pages[min(j, r.kv_len - 1) >> kv.page_shift];
        const bool block_bad = page < 0 || page >= p.num_pages;
        bad_next = __ballot_sync(0xffffffffu, block_bad) & ((1u << kBlocks) - 1u);
        if (block_bad) {
          if (j < r.kv_len) atomicCAS(p.err, 0u, (unsigned)kDevErrBadIndex);
          page = 0;
        }
      };
      uint4 k_code[S::kPieces], v_code[S::kPieces];
      unsigned short k_scale = 0, v_scale = 0;
      const int scale_key = t / S::kGroups, scale_group = t % S::kGroups;
      const unsigned char *k_base = kv.k_codes + piece * 16, *v_base = kv.v_codes + piece * 16;
      const unsigned head_at = (unsigned)head << kv.page_shift;
      auto fetch = [&](uint4 (&code)[S::kPieces], const unsigned char* from, unsigned stride, int j0) {
        #pragma unroll
        for (int i = 0; i < S::kPieces; ++i) {
          const unsigned g = (unsigned)__shfl_sync(0xffffffffu, page, i * (kRowStep / 16) + (row >> 4));
          const unsigned at = head_at + ((j0 + row + i * kRowStep) & in_page);
          code[i] = *reinterpret_cast<const uint4*>(from + (unsigned long long)g * stride + (unsigned long long)at * S::kRowBytes);
        }
      };
      auto fetch_keys = [&](int j0) {
        bad = bad_next;
        fetch(k_code, k_base, kv.k_page, j0);
        const unsigned g = (unsigned)__shfl_sync(0xffffffffu, page, scale_key >> 4);
        const unsigned at = (head_at + ((j0 + scale_key) & in_page)) * S::kGroups + scale_group;
        k_scale = kv.k_scales[(unsigned long long)g * kv.ks_page + at];
        v_scale = kv.v_scales[(unsigned long long)g * kv.vs_page + at];
      };
      auto fetch_values = [&](int j0) { fetch(v_code, v_base, kv.v_page, j0); };
      // Where the thread's first piece goes in a stage: a later one lies kRowStep rows, the same swizzle, further on.
      // Lanes of the odd atoms begin with the second run of results: eight lanes then write eight different banks.
      const int flip = BITS == 8 ? piece >> 2 & 1 : 0;
      uint32_t place[S::kPerPiece / 8];
      #pragma unroll
      for (int c = 0; c < S::kPerPiece / 8; ++c) {
        const int d = piece * S::kPerPiece + (c ^ flip) * 8;
        place[c] = (uint32_t)((d >> 6) * S::kKeys * 128 + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4));
      }
      // a piece's elements, 8 to 16 bytes, to their places in a swizzled stage
      auto store = [&](uint8_t* stage, int i, const uint4& code) {
        const uint32_t words[4] = {code.x, code.y, code.z, code.w};
        #pragma unroll
        for (int c = 0; c < S::kPerPiece / 8; ++c) {                   // 16-byte runs of results
          uint4 v;
          if constexpr (BITS == 8) {
            const uint32_t x = c ^ flip ? words[2] : words[0], y = c ^ flip ? words[3] : words[1];
            if constexpr (kBf16) {
              att::dec8_b(x, v.x, v.y);
              att::dec8_b(y, v.z, v.w);
            } else {
              dec_w8(x, v.x, v.y);
              dec_w8(y, v.z, v.w);
            }
          } else {
            const uint32_t x = words[c];
            if constexpr (kBf16) {
              // 16-bit lanes with nibbles 2 i and 2 i + 1 at the bottom; 0x430n is 128 + n
              const uint32_t y = x >> 4;
              const uint32_t w0 = __byte_perm(x, y, 0x4400), w1 = __byte_perm(x, y, 0x5511), w2 = __byte_perm(x, y, 0x6622),
                             w3 = __byte_perm(x, y, 0x7733);
              v.x = att::b2_sub(lop3_and_or(w0, 0x000F000Fu, 0x43004300u), 0x43084308u);
              v.y = att::b2_sub(lop3_and_or(w1, 0x000F000Fu, 0x43004300u), 0x43084308u);
              v.z = att::b2_sub(lop3_and_or(w2, 0x000F000Fu, 0x43004300u), 0x43084308u);
              v.w = att::b2_sub(lop3_and_or(w3, 0x000F000Fu, 0x43004300u), 0x43084308u);
            } else {
              dec_w4_adjacent(x, v.x, v.y, v.z, v.w);
            }
          }
          *reinterpret_cast<uint4*>(stage + place[c] + i * kRowStep * 128) = v;
        }
      };
      if (steps > 0) {
        fetch_pages(j_begin);
        fetch_keys(j_begin);
        fetch_values(j_begin);
      }
      for (int i = 0; i < steps; ++i) {
        const int n = step + i, st = n % S::kStages, j0 = j_begin + i * S::kKeys;
        const uint32_t before = (uint32_t)(n / S::kStages - 1);        // parity of the stage's last use
        if (i + 1 < steps) fetch_pages(j0 + S::kKeys);
        if (n >= S::kStages) wait(k_free + st, before, kDevErrEmptyWait);
        #pragma unroll
        for (int q = 0; q < S::kPieces; ++q) store(sm_k + st * S::kStepBytes, q, k_code[q]);
        Slot& slot = slots[n % S::kSlots];
        const bool scale_live = j0 + scale_key < r.kv_len && !(bad >> (scale_key >> 4) & 1);
        const float v_sc = scale_live ? kvc::bf16_bits_to_f(v_scale) : 0.f;
        slot.k[scale_group * S::kKeys + scale_key] = scale_live ? kvc::bf16_bits_to_f(k_scale) * p.scale_log2 : 0.f;
        slot.v[scale_group * S::kKeys + scale_key] = v_sc;
        // zero, negative or not finite: as the least
        float v_log = v_sc > 0.f && v_sc < INFINITY ? fminf(fmaxf(log2f(v_sc), kLeast), kMost) : kLeast;
        #pragma unroll
        for (int o = 1; o < S::kGroups; o <<= 1) v_log = fmaxf(v_log, __shfl_xor_sync(0xffffffffu, v_log, o));
        if (scale_group == 0) slot.v_log[scale_key] = v_log;
        const unsigned bits = __float_as_uint(v_sc);
        const unsigned top = __reduce_max_sync(0xffffffffu, bits < 0x7F800000u ? bits : 0u);
        if (lane == 0) slot.v_top[t >> 5] = top;
        if (t == 0) slot.bad = bad;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(k_full + st);
        if (i + 1 < steps) fetch_keys(j0 + S::kKeys);
        if (n >= S::kStages) wait(v_free + st, before, kDevErrEmptyWait);
        #pragma unroll
        for (int q = 0; q < S::kPieces; ++q) store(sm_v + st * S::kStepBytes, q, v_code[q]);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full + st);
        if (i + 1 < steps) fetch_values(j0 + S::kKeys);
      }
      end_segment(g);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmaxRegisters));
    while (u < u_end) {
      // ------------------------------------------------------------- softmax
      const Segment g = next_segment();
      const int steps = g.steps, head = g.head, j_begin = g.j_begin, row0 = g.row0, rows = g.rows;
      const int k_begin = g.k_begin, per_item = g.per_item;
      const int w = warp >> 2, quarter = warp & 3;
      const int local = w * kTileRows + quarter * 32 + lane;           // row of the item
      const bool live = local < rows;
      const int token = live ? p.by_group.of(row0 + local) : 0;
      const int qh = head * p.group + (live ? row0 + local - token * p.group : 0);
      const bool active = w == 0 || g.pair;
      // the warp's 32 rows of queries into shared memory, neighbouring lanes at neighbouring addresses
      if (active && steps > 0) {
        constexpr int kChunks = D / 8, kAhead = 8;                     // loads on their way at a time
        #pragma unroll 1
        for (int i0 = 0; i0 < kChunks; i0 += kAhead) {
          uint4 v[kAhead];
          #pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const int at = w * kTileRows + quarter * 32 + ((i0 + i) * 32 + lane) / kChunks, c = lane % kChunks;
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (at < rows) {
              const int tok = p.by_group.of(row0 + at), h = head * p.group + row0 + at - tok * p.group;
              const kvc::Chunk k = {c * 8, c * 8 + 4, false};
              v[i] = kvc::load_chunk(static_cast<const T*>(p.q.p) + (long long)(r.q0 + tok) * p.q.token_stride + h * p.q.head_stride,
                                     k, p.q.vec);
            }
          }
          #pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const int at = quarter * 32 + ((i0 + i) * 32 + lane) / kChunks, c = lane % kChunks;
            *reinterpret_cast<uint4*>(sm_q + ((w * S::kAtoms + (c >> 3)) * kTileRows + at) * 128 + (((c & 7) ^ (at & 7)) << 4)) = v[i];
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      gemm::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);

      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const uint32_t s_at = tmem + lanes + (uint32_t)(w * 128), o_at = tmem + lanes + (uint32_t)(256 + w * D);
      // Weights are 2^(score - ref).  What is multiplied is a weight times its value's scale, and ref is put where the
      // row's largest such product is 2^kAim, so that in fp16 it is the small ones beside it that lose bits, whatever the
      // scales are.  A step's weights are taken with the reference as it is, half a step at a time, and only where a
      // product could pass 2^kCap (an overflow too) does it move, by a whole number where it can, so that the outputs
      // follow exactly.  (At 4 bits a key's groups share its weight: one whose scales are all 2^-20 of the other's and
      // less loses bits in fp16.)
      float ref = 0.f, sum = 0.f;
      for (int i = 0; i < steps && active; ++i) {
        const int n = step + i, j0 = j_begin + i * S::kKeys;
        const Slot& slot = slots[n % S::kSlots];
        wait(s_full + w, tile_steps + i, kDevErrFullWait);
        gemm::tc_fence_after();
        const unsigned bad = slot.bad;
        const bool some_hidden = bad != 0 || j0 + S::kKeys > att::context_of<SHARED>(p, r);
        const float v_top = fminf(fmaxf(__uint_as_float(max(max(slot.v_top[0], slot.v_top[1]), max(slot.v_top[2], slot.v_top[3]))),
                                        att::pow2((int)kLeast)), att::pow2((int)kMost));
        // the 32 positions of run c that the row sees, as bits
        auto seen = [&](int c) {
          unsigned see = live ? sees32<SHARED>(p, r, token, j0 + c * 32) : 0u;
          if (bad >> (2 * c) & 1) see &= 0xFFFF0000u;
          if (bad >> (2 * c + 1) & 1) see &= 0x0000FFFFu;
          return see;
        };
        // f = the 32 scores of run c less `less`, in units of log2.  (hidden: some of the step's positions are hidden
        // from some row; always a constant.  Two bodies: a branch around the selections within one becomes as many
        // predicated ones that every step executes, 30 of 176 us.)
        auto scores = [&](bool hidden, float (&f)[32], int c, float less, unsigned see) __attribute__((always_inline)) {
          uint32_t x[32], y[32];
          tmem_ld32(s_at + (uint32_t)(c * 32), x);
          if constexpr (S::kGroups > 1) tmem_ld32(s_at + (uint32_t)(S::kKeys + c * 32), y);
          tmem_wait(x);
          if constexpr (S::kGroups > 1) tmem_wait(y);
          #pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 k = *reinterpret_cast<const float4*>(&slot.k[c * 32 + e]);
            F2 a = fma2({__uint_as_float(x[e]), __uint_as_float(x[e + 1])}, {k.x, k.y}, {-less, -less});
            F2 b = fma2({__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])}, {k.z, k.w}, {-less, -less});
            if constexpr (S::kGroups > 1) {
              const float4 l = *reinterpret_cast<const float4*>(&slot.k[S::kKeys + c * 32 + e]);
              a = fma2({__uint_as_float(y[e]), __uint_as_float(y[e + 1])}, {l.x, l.y}, a);
              b = fma2({__uint_as_float(y[e + 2]), __uint_as_float(y[e + 3])}, {l.z, l.w}, b);
            }
            f[e] = a.x;
            f[e + 1] = a.y;
            f[e + 2] = b.x;
            f[e + 3] = b.y;
          }
          if (hidden) {
            #pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(see >> e & 1)) f[e] = -INFINITY;
          }
        };
        // log2 of the largest weight times value scale of runs c .. c + n - 1, less `less`
        auto most = [&](int c, int n, float less) {
          float top = -INFINITY;
          #pragma unroll 1
          for (; n > 0; --n, ++c) {
            float f[32];
            scores(true, f, c, less, seen(c));
            #pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 v = *reinterpret_cast<const float4*>(&slot.v_log[c * 32 + e]);
              f[e] += v.x;
              f[e + 1] += v.y;
              f[e + 2] += v.z;
              f[e + 3] += v.w;
            }
            float a = fmaxf(f[0], f[1]), b = fmaxf(f[2], f[3]);
            #pragma unroll
            for (int e = 4; e < 32; e += 4) {
              a = fmaxf(a, fmaxf(f[e], f[e + 1]));
              b = fmaxf(b, fmaxf(f[e + 2], f[e + 3]));
            }
            top = fmaxf(top, fmaxf(a, b));
          }
          return top;
        };
        // sum and outputs times 2^by, by <= 0, in two factors: what is left may be a normal number where 2^by is none
        auto lower = [&](float by, bool outputs) {
          const float f0 = att::ex2<false>(fmaxf(by, -100.f)), f1 = att::ex2<false>(fminf(by + 100.f, 0.f));
          sum = sum * f0 * f1;
          if (!outputs) return;
          #pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t x[32], y[16];
            tmem_ld32(o_at + (uint32_t)(c * 32), x);
            tmem_wait(x);
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
              #pragma unroll
              for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(x[16 * h + e]) * f0 * f1);
              tmem_st16(o_at + (uint32_t)(c * 32 + 16 * h), y);
            }
          }
        };
        if (__any_sync(0xffffffffu, live && !(sum > 0.f))) {            // rows that have seen nothing yet
          const float top = most(0, S::kKeys / 32, 0.f);
          // (rounded down: a score of 2^23 and more that came out too high would leave its row without weight)
          if (!(sum > 0.f) && top > -INFINITY) ref = top - kAim - fabsf(top) * 0x1p-22f;
        }
        // the weights of half h, in the place of its scores
        constexpr int kRuns = S::kKeys / 64;                           // of 32 scores
        auto weigh_half = [&](bool hidden, int h) __attribute__((always_inline)) {
          float part;
          uint32_t hi[kRuns][S::kGroups][16], lo[kRuns][S::kGroups][16];
          auto weigh = [&](bool moved) __attribute__((always_inline)) {
            F2 sums[2] = {{0.f, 0.f}, {0.f, 0.f}};
            #pragma unroll
            for (int i32 = 0; i32 < kRuns; ++i32) {
              const int c = h * kRuns + i32;
              const unsigned see = hidden ? seen(c) : 0xFFFFFFFFu;
              float f[32];
              scores(hidden, f, c, ref, see);
              if (moved) {                                             // what the reference cannot follow (below)
                #pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float cap = kCap - slot.v_log[c * 32 + e];
                  f[e] = f[e] > cap ? cap : f[e];
                }
              }
              #pragma unroll
              for (int e = 0; e < 32; ++e) f[e] = att::ex2<kBf16>(f[e]);
              #pragma unroll
              for (int e = 0; e < 32; e += 4) {
                sums[0] = add2(sums[0], {f[e], f[e + 1]});
                sums[1] = add2(sums[1], {f[e + 2], f[e + 3]});
              }
              #pragma unroll
              for (int q = 0; q < S::kGroups; ++q)
                #pragma unroll
                for (int e = 0; e < 32; e += 4) {
                  const float4 v = *reinterpret_cast<const float4*>(&slot.v[q * S::kKeys + c * 32 + e]);
                  F2 a[2] = {mul2({f[e], f[e + 1]}, {v.x, v.y}), mul2({f[e + 2], f[e + 3]}, {v.z, v.w})};
                  if (hidden) {                                        // whatever a hidden value's scale is
                    if (!(see >> e & 1)) a[0].x = 0.f;
                    if (!(see >> (e + 1) & 1)) a[0].y = 0.f;
                    if (!(see >> (e + 2) & 1)) a[1].x = 0.f;
                    if (!(see >> (e + 3) & 1)) a[1].y = 0.f;
                  }
                  #pragma unroll
                  for (int g2 = 0; g2 < 2; ++g2) {
                    if constexpr (kBf16) {
                      const uint32_t u2 = att::pack_b2(a[g2].x, a[g2].y);
                      hi[i32][q][e / 2 + g2] = u2;
                      lo[i32][q][e / 2 + g2] =
                          att::pack_b2(a[g2].x - __uint_as_float(u2 << 16), a[g2].y - __uint_as_float(u2 & 0xFFFF0000u));
                    } else {
                      hi[i32][q][e / 2 + g2] = att::pack_h2(a[g2].x, a[g2].y);
                    }
                  }
                }
            }
            part = (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
          };
          weigh(false);
          const bool over = part * v_top > att::pow2((int)kCap);
          if (__any_sync(0xffffffffu, over)) {                         // the scores are still there
            const float top = most(h * kRuns, kRuns, ref);
            // A reference of 2^23 and more has no room for whole numbers.  It then stays below the largest product by
            // what the two may be off, and what is beyond the cap, of scores equal to the last bits, becomes the cap's.
            const float by_most = over && top < INFINITY ? ceilf(top - kAim - (fabsf(ref) + fabsf(top)) * 0x1p-22f) : 0.f;
            const float moved = __fadd_rd(ref, fmaxf(by_most, 0.f)), by = moved - ref;
            if (h > 0) wait(half_done + w, tile_steps + i, kDevErrFullWait);   // the first half is in the outputs
            gemm::tc_fence_after();
            lower(-by, i > 0 || h > 0);
            ref = moved;
            weigh(true);
          }
          sum += part;
          #pragma unroll
          for (int i32 = 0; i32 < kRuns; ++i32)
            #pragma unroll
            for (int q = 0; q < S::kGroups; ++q) {
              const uint32_t at = s_at + (uint32_t)(q * S::kKeys + (h * kRuns + i32) * 32);
              tmem_st16(at, hi[i32][q]);
              if constexpr (kBf16) tmem_st16(at + 16u, lo[i32][q]);
            }
          gemm::tmem_st_wait();
          gemm::tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_ready + 2 * w + h);
        };
        #pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          if (some_hidden)
            weigh_half(true, h);
          else
            weigh_half(false, h);
        }
      }
      wait(o_done, segment, kDevErrFullWait);
      gemm::tc_fence_after();
      if (!(sum != 0.f)) ref = att::kLow;                              // nothing seen (a NaN sum stays one)

      // ------------------------------------------------- outputs, or a part
      const long long item_begin = g.item_begin;
      const bool whole = k_begin == 0 && g.k_end == per_item;
      const long long out_at = (long long)(r.q0 + token) * p.q_heads + qh;
      auto finish = [&](int c, const float (&o)[32], float top, float l) {     // 32 outputs of the row
        if (!live) return;
        float now = 1.f, then = 0.f;                        // what the two passes' outputs are taken with
        if constexpr (SHARED) {
          float4* early = reinterpret_cast<float4*>(p.early_out + out_at * D + c * 32);
          if (p.first_pass) {
            #pragma unroll
            for (int e = 0; e < 8; ++e) early[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            if (c == 0) p.early_sums[out_at] = make_float2(top, l);
            return;
          }
          const float2 e = p.early_sums[out_at];
          if (e.y != 0.f) {                                 // there is something (a NaN too)
            const float most = fmaxf(top, e.x);
            now = att::ex2<true>(top - most);
            then = att::ex2<true>(e.x - most);
            top = most;
            l = l * now + e.y * then;
          }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        now *= inv;
        then *= inv;
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + out_at * D + c * 32);
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float* f = o + 8 * e;
          float more[8] = {};
          if (SHARED && then != 0.f) {
            const float4* early = reinterpret_cast<const float4*>(p.early_out + out_at * D + c * 32 + 8 * e);
            const float4 x = early[0], y = early[1];
            const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            #pragma unroll
            for (int i = 0; i < 8; ++i) more[i] = v[i] * then;
          }
          uint32_t words[4];
          #pragma unroll
          for (int i = 0; i < 4; ++i)
            words[i] = SHARED ? kvc::pack2<T>(fmaf(f[2 * i], now, more[2 * i]), fmaf(f[2 * i + 1], now, more[2 * i + 1]))
                              : kvc::pack2<T>(f[2 * i] * now, f[2 * i + 1] * now);
          dst[e] = make_uint4(words[0], words[1], words[2], words[3]);
        }
        if (p.lse && c == 0) p.lse[out_at] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.69314718056f;
      };
      // a part: [reference][sum] of the rows, then runs of 4 outputs of all rows one behind another
      auto park = [&](float* dst, int c, const float (&o)[32], float top, float l) {
        if (!live) return;
        #pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<float4*>(dst + 2 * kRows + ((c * 8 + e) * kRows + local) * 4) =
              make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        if (c == 0) {
          dst[local] = top;
          dst[kRows + local] = l;
        }
      };
      float* mine_out = partials + (long long)(2 * blockIdx.x + (k_begin == 0)) * S::kPartial;
      if (active) {
        #pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t x[32] = {};
          float o[32];
          if (steps > 0) {
            tmem_ld32(o_at + (uint32_t)(c * 32), x);
            tmem_wait(x);
          }
          #pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(x[e]);
          if (whole)
            finish(c, o, ref, sum);
          else
            park(mine_out, c, o, ref, sum);
        }
      }
      if (!whole && !(SHARED && p.first_pass)) {            // those of a first pass are joined by att::join_kernel
        const att::Join j = att::join_of(work, item_begin, per_item, (int)blockIdx.x);
        auto part = [&](int q) {                            // the first begins the item: its CTA's second slot
          return partials + (long long)(2 * (j.c_first + q) + (q == 0)) * S::kPartial;
        };
        auto arrive = [&](unsigned* counter, int n) {       // true in the last of n CTAs, which sees the others' parts
          __threadfence();
          named_bar_sync(1, 32 * kSoftmaxWarps);
          if (threadIdx.x == 0) {
            *last_one = atomic_add_acq_rel_gpu(counter, 1u) == (unsigned)n - 1;
            if (*last_one) *counter = 0;
          }
          named_bar_sync(1, 32 * kSoftmaxWarps);
          return *last_one != 0;
        };
        // a thread joins its own row, and no other reads the row's parts
        auto join = [&](int first, int stride, int count, auto out) {
          float top = att::kLow, l = 0.f;
          for (int q = 0; q < count; ++q) top = fmaxf(top, __ldcg(part(first + q * stride) + local));
          for (int q = 0; q < count; ++q) {
            const float* src = part(first + q * stride);
            l += __ldcg(src + kRows + local) * att::ex2<true>(__ldcg(src + local) - top);
          }
          float f0 = 0.f;                                   // of the part that `out` may write over: read before
          f0 = att::ex2<true>(__ldcg(part(first) + local) - top);
          #pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32] = {};
            for (int q = 0; q < count; ++q) {
              const float* src = part(first + q * stride);
              const float f = q == 0 ? f0 : att::ex2<true>(__ldcg(src + local) - top);
              #pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 v = __ldcg(reinterpret_cast<const float4*>(src + 2 * kRows + ((c * 8 + e) * kRows + local) * 4));
                o[4 * e] = fmaf(v.x, f, o[4 * e]);
                o[4 * e + 1] = fmaf(v.y, f, o[4 * e + 1]);
                o[4 * e + 2] = fmaf(v.z, f, o[4 * e + 2]);
                o[4 * e + 3] = fmaf(v.w, f, o[4 * e + 3]);
              }
            }
            out(c, o, top, l);
          }
        };
        bool last = true;
        if (j.grouped()) {
          last = arrive(counters + j.group_counter(), j.group_parts);
          if (last && live)
            join(j.group * att::kJoin, 1, j.group_parts, [&](int c, const float (&o)[32], float top, float l) {
              park(part(j.group * att::kJoin), c, o, top, l);
            });
        }
        if (last && arrive(counters + j.item_counter(), j.item_arrivals()) && live)
          join(0, j.groups > 1 ? att::kJoin : 1, j.item_arrivals(), finish);
      }
      if (active) tile_steps += steps;
      end_segment(g);
    }
  }

  gemm::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    gemm::tc_fence_after();
    gemm::tmem_dealloc(tmem, 512);
  }
}

// A first pass's parts, for att::join_kernel.
template <int D, int BITS>
struct TreePart {
  static constexpr int kRows = tree::kRows, kUnits = kMinUnits, kFloats = Shape<D, BITS>::kPartial;
  static constexpr bool kLanesAreRows = true;
  static __device__ __forceinline__ int at(int row, int place) { return 2 * kRows + (place / 4 * kRows + row) * 4; }
  static __device__ __forceinline__ int element(int place) { return place; }
};

}  // namespace tree
}  // namespace ql
