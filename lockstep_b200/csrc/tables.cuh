// A step's tables from its request lengths: query starts, slots, positions, and the pages that new
// tokens need, taken from a free list in sequence order.
//
// Integer work of a few hundred KB at most, so launches and dependent passes are what costs.  One
// launch: every CTA scans all n lengths itself (a few us at n = 1,000, from L2) instead of waiting for
// another CTA's scan, keeps both prefix sums in shared memory, and then writes its share of the block
// table and of the token arrays.  A token's page is computed from the free list, not read back from the
// table row that another CTA may be writing; only the page that was open before the step is read, and
// no CTA writes that one.
#pragma once
#include "common.cuh"

namespace lssab8 {

constexpr int kTblThreads = 1024;
constexpr int kTblMaxSeqs = 16384;                           // three 4-byte arrays of n in shared memory
constexpr int kTblMaxTokens = 1 << 30;                       // 32-bit token counters step past it by a grid's threads

struct TablesArgs {
  const int32_t *before, *fresh;      // [n] lengths before the step, new tokens
  int n, max_pages, nfree, cap;       // cap: length of the token arrays
  int32_t* table;                     // [n, max_pages], updated in place
  long long table_stride;
  const int32_t* free_pages;          // [nfree]
  int32_t *qsl, *after, *seq_index, *used;   // [n + 1], [n], [cap], [1]
  long long *slots, *positions;       // [cap]
  int* err;
};

// exclusive scan of one (tokens, pages) pair a thread over the CTA, 64-bit: (sums before, total)
__device__ __forceinline__ void scan_pair(long long& a, long long& b, long long& ta, long long& tb, long long (*ws)[32]) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const long long a0 = a, b0 = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) { a += x; b += y; }
  }
  if (lane == 31) { ws[0][w] = a; ws[1][w] = b; }
  __syncthreads();
  long long pa = 0, pb = 0;
  ta = 0; tb = 0;
  for (int i = 0; i < nw; ++i) {
    if (i < w) { pa += ws[0][i]; pb += ws[1][i]; }
    ta += ws[0][i]; tb += ws[1][i];
  }
  __syncthreads();
  a += pa - a0;
  b += pb - b0;
}

__global__ void __launch_bounds__(kTblThreads) step_tables_kernel(const TablesArgs p) {
  extern __shared__ int32_t sm[];
  int32_t* start = sm;                 // [n + 1] first token of a sequence
  int32_t* page0 = sm + p.n + 1;       // [n + 1] first free-list entry of a sequence
  int32_t* len0 = sm + 2 * (p.n + 1);  // [n]
  __shared__ long long ws[2][32];
  const int tid = threadIdx.x;
  const int per = (p.n + kTblThreads - 1) / kTblThreads;     // consecutive sequences a thread
  const int i0 = min(tid * per, p.n), i1 = min(i0 + per, p.n);
  bool bad = false;
  long long tok = 0, pg = 0, ttok, tpg;
  auto lens = [&](int i, int& b, int& m) {                   // lengths below 0 or above 2^30 count as 0
    b = p.before[i];
    m = p.fresh[i];
    if (b < 0 || m < 0 || (long long)b + m > (1 << 30)) { b = 0; m = 0; bad = true; }
  };
  for (int i = i0; i < i1; ++i) {
    int b, m;
    lens(i, b, m);
    tok += m;
    pg += pages_of(b + m) - pages_of(b);
  }
  scan_pair(tok, pg, ttok, tpg, ws);
  constexpr long long kMax = 0x7FFFFFFFll;
  for (int i = i0; i < i1; ++i) {
    int b, m;
    lens(i, b, m);
    start[i] = (int)min(tok, kMax);
    page0[i] = (int)min(pg, kMax);
    len0[i] = b;
    tok += m;
    pg += pages_of(b + m) - pages_of(b);
  }
  if (tid == 0) { start[p.n] = (int)min(ttok, kMax); page0[p.n] = (int)min(tpg, kMax); }
  __syncthreads();
  if (ttok > p.cap || tpg > p.nfree) bad = true;
  if (blockIdx.x == 0) {
    for (int i = tid; i <= p.n; i += kTblThreads) p.qsl[i] = start[i];
    for (int i = tid; i < p.n; i += kTblThreads) p.after[i] = len0[i] + (start[i + 1] - start[i]);
    if (tid == 0) p.used[0] = (int)min(tpg, (long long)p.nfree);
  }
  const int gid = blockIdx.x * kTblThreads + tid, gsz = gridDim.x * kTblThreads;
  // the sequence of an entry of a prefix sum: the last i with first[i] <= x
  auto find = [&](const int32_t* first, int x) {
    int lo = 0, hi = p.n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
  };
  const int take = min(page0[p.n], p.nfree);
  for (long long x = gid; x < take; x += gsz) {              // the pages this step takes (a list may reach 2^31)
    const int e = (int)x, i = find(page0, e);
    const int j = pages_of(len0[i]) + (e - page0[i]);
    if (j < p.max_pages) p.table[i * p.table_stride + j] = p.free_pages[e];
    else bad = true;
  }
  for (int t = gid; t < p.cap; t += gsz) {
    long long slot = -1, pos = 0;
    int seq = -1;
    if (t < start[p.n]) {
      seq = find(start, t);
      pos = (long long)len0[seq] + (t - start[seq]);
      const int j = (int)(pos >> 4), have = pages_of(len0[seq]);
      int page = -1;
      if (j < p.max_pages) {
        const long long e = (long long)page0[seq] + j - have;
        if (j < have) page = p.table[seq * p.table_stride + j];
        else if (e < p.nfree) page = p.free_pages[e];
      }
      if (page >= 0) slot = (long long)page * 16 + (pos & 15);
      else bad = true;
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
    p.seq_index[t] = seq;
  }
  if (bad) atomicOr(p.err, kDevPlan);
}

}  // namespace lssab8
