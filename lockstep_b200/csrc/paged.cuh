// Attention over the paged lattice for whole steps: the plan of the packed prompt rows.  (Their kernel,
// and the shared-prefix kernel, are prefill_kernel's paged forms, prefill.cuh; a shared batch's own
// blocks and refold are the decode kernels' SHARED forms.)
#pragma once
#include "common.cuh"

namespace lssab8 {

constexpr int kRowsPlanThreads = 1024;
constexpr int kRowsPlanBins = 2048;

struct RowsPlanArgs {
  const int32_t* cu_q;          // [B + 1] first row of each sequence
  const int32_t* seq_lens;      // [B]
  const int32_t* prefix;        // [B] or nullptr
  const uint8_t* active;        // [B] or nullptr: sequences with 0 have no rows here
  int B, N, max_blocks, max_pages;
  int* tile_off;                // [B + 1]
  int4* tiles;                  // [max_tiles], max_tiles = N / 128 + B: enough for rows that do not overlap
  int max_tiles;
  int* ntiles;
  int* err;
};

// The tiles of a step: sequence b's rows are its last n_b = cu_q[b + 1] - cu_q[b] positions, cut into
// 128-row tiles at its own 128-key blocks (its first row is on a block boundary).  Sorted by their
// number of key blocks, longest first, so that the snake order balances the CTAs: a counting sort in
// shared memory; tiles of equal length fall in any order, which changes no result.  A sequence whose
// rows do not fit (off the 128 grid, more rows than keys, a prefix past its end, past the lattice
// arrays) gets no tiles and sets a device error.
__global__ void __launch_bounds__(kRowsPlanThreads) rows_plan_kernel(const RowsPlanArgs p) {
  __shared__ int ws[32];
  __shared__ int carry;
  __shared__ int bins[kRowsPlanBins];
  pdl_launch_dependents();                       // the query quantiser runs beside the plan
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  auto rows_of = [&](int b, int& n, int& T0, int& P) -> bool {
    n = 0;
    if (p.active && !p.active[b]) return true;
    const int c0 = p.cu_q[b], c1 = p.cu_q[b + 1], L = p.seq_lens[b];
    if (c0 == c1) return true;
    P = p.prefix ? p.prefix[b] : 0;
    if (c0 < 0 || c1 < c0 || c1 > p.N || L < c1 - c0 || ((L - (c1 - c0)) & (kKB - 1)) || P < 0 || P > L) return false;
    n = c1 - c0;
    T0 = L - n;
    return true;
  };
  if (tid == 0) carry = 0;
  for (int i = tid; i < kRowsPlanBins; i += kRowsPlanThreads) bins[i] = 0;
  __syncthreads();
  for (int base = 0; base < p.B; base += kRowsPlanThreads) {
    const int b = base + tid;
    int nt = 0;
    if (b < p.B) {
      int n, T0, P;
      if (!rows_of(b, n, T0, P)) atomicOr(p.err, kDevPlan);
      else if (n > 0) {
        const int L = p.seq_lens[b];
        if ((L + kKB - 1) / kKB > p.max_blocks || (L + 15) / 16 > p.max_pages) atomicOr(p.err, kDevBadPage);
        else nt = (n + 127) / 128;
      }
    }
    int x = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) ws[w] = x;
    __syncthreads();
    int before = carry, all = 0;
    for (int i = 0; i < 32; ++i) {
      if (i < w) before += ws[i];
      all += ws[i];
    }
    if (b < p.B) p.tile_off[b] = before + x - nt;
    __syncthreads();
    if (tid == 0) carry += all;
    __syncthreads();
  }
  if (tid == 0 && carry > p.max_tiles) atomicOr(p.err, kDevPlan);     // overlapping rows (cu_q not ascending)
  const int total = min(carry, p.max_tiles);
  if (tid == 0) { p.tile_off[p.B] = total; *p.ntiles = total; }
  __syncthreads();                               // (one CTA: its own writes to tile_off are visible)
  auto tile_at = [&](int e, int& key) -> int4 {
    int lo = 0, hi = p.B;                        // the sequence: the last b with tile_off[b] <= e
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.tile_off[mid] <= e) lo = mid; else hi = mid;
    }
    int n, T0 = 0, P = 0;
    rows_of(lo, n, T0, P);
    const int t = e - p.tile_off[lo];
    const int kt = T0 / kKB + t;
    int nb = kt + 1;
    if (kt * kKB < P) nb = max(nb, (P + kKB - 1) / kKB);
    key = kRowsPlanBins - min(nb, kRowsPlanBins);      // longest first
    return make_int4(lo, kt, nb, p.cu_q[lo] + t * 128);
  };
  for (int e = tid; e < total; e += kRowsPlanThreads) {
    int key;
    tile_at(e, key);
    atomicAdd(&bins[key], 1);
  }
  __syncthreads();
  // exclusive scan of the bins, two a thread
  const int a = bins[2 * tid], c = bins[2 * tid + 1];
  int x = a + c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) ws[w] = x;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < w; ++i) before += ws[i];
  bins[2 * tid] = before + x - a - c;
  bins[2 * tid + 1] = before + x - c;
  __syncthreads();
  for (int e = tid; e < total; e += kRowsPlanThreads) {
    int key;
    const int4 t = tile_at(e, key);
    p.tiles[atomicAdd(&bins[key], 1)] = t;
  }
}

}  // namespace lssab8
