// qplan.cuh — a serving step's page tables, slots and positions from request
// lengths, on the GPU (sm_100a).
//
// With P = page size, a request that holds lens tokens, keeps `keep` of them
// and grows by `fresh` new ones
//   held = ceil(lens / P), kept = ceil(keep / P), need = ceil((keep + fresh) / P)
// gives held - kept pages back and takes need - kept.  Free pages are a stack.
// The pages that come back, in the order of requests and positions, are pushed
// so that the first of them lies on top; then pages are taken from the top in
// the same order.  Cutting off and growing by as much therefore restores a
// request's own pages.  New token t of request b is at position keep + t, in
// slot page * P + position % P.
//
// A request is served if its pages fit its table row, the new tokens up to and
// with its own fit the step, and either it takes no page or the pages taken up
// to and with its own are there: one that waits for pages is not overtaken by
// one behind it that needs some.  A request that is not served is cut to what
// it keeps, and gets no new tokens.
//
// All of it is prefix sums over the requests, then one lookup a token.  What
// bounds it is a chain of latencies: the lengths' way from memory, three scans,
// the pages' way; so one launch does everything.  Many requests are scanned by
// each CTA of a cluster for itself (nothing has to be handed over), and a barrier
// of the cluster separates the reading of the old state from the writing of the
// new.  Many tokens (12 bytes each to be written, more than a cluster's SMs write
// quickly) are left to a second kernel over all SMs, which looks them up in the
// tables as they then are.
//
// One request: 3.7 us; 64 requests with trees (2100 tokens) 7.0; 1000 requests, 5900 tokens: 10.7 (one kernel: 12.9); 23
// prompts, 131000 tokens: 10.7 (by the cluster's SMs alone: 23), of which the tokens' writes need 0.4.
#pragma once

#include "ql_common.cuh"

namespace ql {
namespace plan {

constexpr int kMaxBatch = 8192;
constexpr int kThreads = 1024, kWarps = kThreads / 32;

struct Params {
  int* table;                      // [batch][table_stride]
  int* lens;                       // [batch]
  int* stack;                      // [num_pages]: the first *count are free
  int* count;
  const int* keep;                 // [batch], or null: all
  const int* fresh;                // [batch]
  int* cu_q;                       // [batch + 1]
  long long* slots;                // [max_tokens]
  int* positions;                  // [max_tokens]
  int* refused;
  long long table_stride, max_tokens;
  int batch, width, num_pages, page_shift;
  bool tokens;                     // the first kernel looks them up
};

struct Request {
  int lens, keep, held, kept;
  unsigned fresh, grow;            // asked for; 0 where the table's row has no room
  bool fits;
};
__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  const long long room = min((long long)p.width << p.page_shift, 0x7FFFFFFFll);
  const long long page = (1 << p.page_shift) - 1;
  r.lens = (int)min((long long)max(p.lens[b], 0), room);
  r.keep = p.keep ? min(max(p.keep[b], 0), r.lens) : r.lens;
  r.held = (int)((r.lens + page) >> p.page_shift);
  r.kept = (int)((r.keep + page) >> p.page_shift);
  const long long want = (long long)r.keep + max(p.fresh[b], 0);
  r.fits = want <= room;
  r.fresh = r.fits ? (unsigned)(want - r.keep) : 0u;
  r.grow = r.fits ? (unsigned)((want + page) >> p.page_shift) - (unsigned)r.kept : 0u;
  return r;
}

// Sums that stop at kMost: more is never asked whether it fits.  (Associative, of what is kMost at most.)
constexpr unsigned kMost = 0x7FFFFFFFu;
__device__ __forceinline__ unsigned plus(unsigned a, unsigned b) { return min(a + b, kMost); }

// Inclusive sums over the CTA's threads, and the CTA's.
template <int N>
__device__ __forceinline__ void scan(unsigned (&v)[N], unsigned (&all)[N], unsigned (*warp_sum)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  #pragma unroll
  for (int o = 1; o < 32; o <<= 1)
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned u = __shfl_up_sync(0xffffffffu, v[i], o);
      if (lane >= o) v[i] = plus(v[i], u);
    }
  __syncthreads();                 // the sums of the scan before have been read
  if (lane == 31)
    #pragma unroll
    for (int i = 0; i < N; ++i) warp_sum[warp][i] = v[i];
  __syncthreads();
  #pragma unroll
  for (int i = 0; i < N; ++i) {
    unsigned s = lane < warps ? warp_sum[lane][i] : 0;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s = plus(s, u);
    }
    all[i] = __shfl_sync(0xffffffffu, s, 31);
    const unsigned before = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
    if (warp > 0) v[i] = plus(v[i], before);
  }
}

// The largest b < n with first[b] <= i, for first[0] = 0 <= i.
__device__ __forceinline__ int holder(const int* first, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Four tokens from t0 on, a multiple of four.
__device__ __forceinline__ void store_tokens(const Params& p, long long t0, const long long (&slot)[4], const int (&position)[4]) {
  if (t0 + 4 <= p.max_tokens) {
    reinterpret_cast<longlong2*>(p.slots + t0)[0] = make_longlong2(slot[0], slot[1]);
    reinterpret_cast<longlong2*>(p.slots + t0)[1] = make_longlong2(slot[2], slot[3]);
    *reinterpret_cast<int4*>(p.positions + t0) = make_int4(position[0], position[1], position[2], position[3]);
  } else {
    for (int i = 0; t0 + i < p.max_tokens; ++i) {
      p.slots[t0 + i] = slot[i];
      p.positions[t0 + i] = position[i];
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1) plan_kernel(const Params p) {
  extern __shared__ int smem[];
  // of each request: its first new token, what it keeps, the first page that it takes, the first that comes back
  int* first_token = smem;
  int* keeps = first_token + p.batch + 1;
  int* first_taken = keeps + p.batch;
  int* first_back = first_taken + p.batch + 1;
  __shared__ unsigned warp_sum[kWarps][2];
  griddep_launch_dependents();
  griddep_wait();
  const int rank = (int)cluster_rank(), ctas = (int)gridDim.x, threads = (int)blockDim.x;
  const long long page_mask = (1 << p.page_shift) - 1;
  const int count = min(max(*p.count, 0), p.num_pages);

  // pages that come back; the requests of the first round stay in registers
  unsigned back = 0;                                          // below 2^31: the table has no more entries
  Request first = {};
  for (int i = 0; i < p.batch; i += threads) {
    const int b = i + (int)threadIdx.x;
    Request r = {};
    if (b < p.batch) r = request(p, b);
    if (i == 0) first = r;
    const unsigned mine = (unsigned)(r.held - r.kept);
    unsigned v[1] = {mine}, all[1];
    scan<1>(v, all, warp_sum);
    if (b < p.batch) {
      keeps[b] = r.keep;
      first_back[b] = (int)(back + v[0] - mine);
    }
    back += all[0];
  }
  // who is served, and what they get
  const long long available = (long long)count + back;
  unsigned asked[2] = {0, 0}, given[2] = {0, 0};
  int refused = 0;
  for (int i = 0; i < p.batch; i += threads) {
    const int b = i + (int)threadIdx.x;
    Request r = first;
    if (i > 0 && b < p.batch) r = request(p, b);
    const bool live = b < p.batch;
    unsigned v[2] = {live ? r.fresh : 0u, live ? r.grow : 0u}, all[2];
    const unsigned fresh = v[0], grow = v[1];
    scan<2>(v, all, warp_sum);
    const bool served = live && r.fits && plus(asked[0], v[0]) <= p.max_tokens && (grow == 0 || plus(asked[1], v[1]) <= available);
    refused += live && !served && p.fresh[b] > 0;
    asked[0] = plus(asked[0], all[0]);
    asked[1] = plus(asked[1], all[1]);
    unsigned w[2] = {served ? fresh : 0u, served ? grow : 0u};
    const unsigned mine[2] = {w[0], w[1]};
    scan<2>(w, all, warp_sum);
    if (live) {
      first_token[b] = (int)(given[0] + w[0] - mine[0]);
      first_taken[b] = (int)(given[1] + w[1] - mine[1]);
    }
    given[0] += all[0];
    given[1] += all[1];
  }
  const int total = (int)given[0], taken = (int)given[1];
  if (threadIdx.x == 0) {
    first_token[p.batch] = total;
    first_taken[p.batch] = taken;
  }
  __syncthreads();

  // pages back onto the stack; several at a time, whose lookups wait together
  constexpr int kAtOnce = 4;
  const int at = rank * threads + (int)threadIdx.x, step = ctas * threads;
  for (long long j0 = at; j0 < back; j0 += (long long)kAtOnce * step) {
    int page[kAtOnce];
    #pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const long long j = j0 + (long long)i * step;
      if (j >= back) continue;
      const int b = holder(first_back, p.batch, (int)j);
      const int k = (int)((keeps[b] + page_mask) >> p.page_shift) + (int)j - first_back[b];
      page[i] = p.table[(long long)b * p.table_stride + k];
    }
    #pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const long long to = available - 1 - (j0 + (long long)i * step);
      if (to >= count && to < p.num_pages) p.stack[to] = page[i];         // to >= count: j < back
    }
  }
  cluster_sync_all();               // the old lengths, count and pages have been read, the stack written
  auto page_taken = [&](int i) {
    const long long from = available - 1 - i;
    return from >= 0 && from < p.num_pages ? p.stack[from] : -1;
  };
  for (long long i0 = at; i0 < taken; i0 += (long long)kAtOnce * step) {
    int page[kAtOnce];
    long long to[kAtOnce];
    #pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const long long n = i0 + (long long)i * step;
      to[i] = -1;
      if (n >= taken) continue;
      const int b = holder(first_taken, p.batch, (int)n);
      to[i] = (long long)b * p.table_stride + (int)((keeps[b] + page_mask) >> p.page_shift) + (int)n - first_taken[b];
      page[i] = page_taken((int)n);
    }
    #pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (to[i] >= 0) p.table[to[i]] = page[i];
  }
  for (int b = at; b <= p.batch; b += step) {
    p.cu_q[b] = first_token[b];
    if (b < p.batch) p.lens[b] = keeps[b] + first_token[b + 1] - first_token[b];
  }
  if (rank == 0) {
    __shared__ int sum;
    if (threadIdx.x == 0) sum = 0;
    __syncthreads();
    if (refused) atomicAdd(&sum, refused);
    __syncthreads();
    if (threadIdx.x == 0) {
      *p.refused = sum;
      *p.count = (int)min(available - taken, (long long)p.num_pages);
    }
  }
  if (!p.tokens) return;
  for (long long t = at; t < p.max_tokens; t += step) {       // one at a time: they are few, and so is the code
    int page = -1, position = 0;
    if (t < total) {
      const int b = holder(first_token, p.batch, (int)t);
      position = keeps[b] + (int)t - first_token[b];
      const int k = position >> p.page_shift, kept = (int)((keeps[b] + page_mask) >> p.page_shift);
      page = k < kept ? p.table[(long long)b * p.table_stride + k] : page_taken(first_taken[b] + k - kept);
    }
    p.slots[t] = page < 0 ? -1 : ((long long)page << p.page_shift) + (position & page_mask);
    p.positions[t] = position;
  }
}

// Slots and positions of four neighbouring tokens a thread, after plan_kernel.
constexpr int kTokenThreads = 256;
__global__ void __launch_bounds__(kTokenThreads) token_kernel(const Params p) {
  griddep_launch_dependents();
  griddep_wait();
  extern __shared__ int cu[];
  for (int i = threadIdx.x; i <= p.batch; i += kTokenThreads) cu[i] = p.cu_q[i];
  __syncthreads();
  const int total = cu[p.batch];
  const long long t0 = 4ll * ((long long)blockIdx.x * kTokenThreads + threadIdx.x);
  if (t0 >= p.max_tokens) return;
  int b = t0 < total ? holder(cu, p.batch, (int)t0) : 0;
  long long slot[4];
  int position[4];
  int first = 0, end = 0, keep = 0;                           // of request b
  if (t0 < total) {
    first = cu[b];
    end = cu[b + 1];
    keep = p.lens[b] - (end - first);
  }
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = (int)t0 + i;
    slot[i] = -1;
    position[i] = 0;
    if (t < total) {
      while (t >= end) {
        first = end;
        end = cu[++b + 1];
        keep = p.lens[b] - (end - first);
      }
      const int pos = keep + t - first;
      const int page = p.table[(long long)b * p.table_stride + (pos >> p.page_shift)];
      slot[i] = page < 0 ? -1 : ((long long)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
      position[i] = pos;
    }
  }
  store_tokens(p, t0, slot, position);
}

}  // namespace plan
}  // namespace ql
