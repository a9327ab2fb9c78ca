// Attention over the paged lattice for whole steps: the plan of the packed prompt rows, and the launch that
// plans a call and quantises its queries.  (Their kernel,
// and the shared-prefix kernel, are prefill_kernel's paged forms, prefill.cuh; a shared batch's own
// blocks and refold are the decode kernels' SHARED forms.)
#pragma once
#include "decode_tc.cuh"
#include "prep.cuh"

namespace lssab8 {

constexpr int kStepPlanThreads = 256;
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
__device__ __forceinline__ void rows_plan(const RowsPlanArgs& p) {
  constexpr int NT = kStepPlanThreads, NW = NT / 32;
  __shared__ int ws[NW];
  __shared__ int carry;
  __shared__ int bins[kRowsPlanBins];
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
  for (int i = tid; i < kRowsPlanBins; i += NT) bins[i] = 0;
  __syncthreads();
  for (int base = 0; base < p.B; base += NT) {
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
    for (int i = 0; i < NW; ++i) {
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
  for (int e = tid; e < total; e += NT) {
    int key;
    tile_at(e, key);
    atomicAdd(&bins[key], 1);
  }
  __syncthreads();
  // exclusive scan of the bins, consecutive ones a thread
  constexpr int PB = kRowsPlanBins / NT;
  int n = 0;
  for (int i = 0; i < PB; ++i) n += bins[PB * tid + i];
  int x = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) ws[w] = x;
  __syncthreads();
  int before = x - n;
  for (int i = 0; i < w; ++i) before += ws[i];
  for (int i = 0; i < PB; ++i) {
    const int c = bins[PB * tid + i];
    bins[PB * tid + i] = before;
    before += c;
  }
  __syncthreads();
  for (int e = tid; e < total; e += NT) {
    int key;
    const int4 t = tile_at(e, key);
    p.tiles[atomicAdd(&bins[key], 1)] = t;
  }
}

// The plan of a call and the query quantiser in one launch: CTA 0 plans, the others quantise rows of q.  (They
// do not read each other; as two kernels the small calls paid one more launch, 4 us of host time.)
struct SharedPlanArgs {
  const int32_t* seq_lens;
  int B, max_blocks, max_pages;
  int *blk_off, *order, *err;
  int shared_blocks;
  int* leader;
};
__device__ __forceinline__ void step_plan(const RowsPlanArgs& p) { rows_plan(p); }
__device__ __forceinline__ void step_plan(const SharedPlanArgs& p) {
  decode_plan<true, kStepPlanThreads>(p.seq_lens, p.B, p.max_blocks, p.max_pages, p.blk_off, p.order, nullptr, 0, p.err,
                                      p.shared_blocks, p.leader);
}
template <typename Plan>
__global__ void __launch_bounds__(kStepPlanThreads) step_plan_kernel(const Plan plan) {
  pdl_launch_dependents();
  step_plan(plan);
}
// P1 over tokens [N, H, dh] (strides 0, token, head; contiguous channels, 16-byte rows): row n H + h of q8 and eq.
// quant_rows_vec's rule with fewer instructions, which bound it here (16,700 tokens of 32 heads: 53 us with its 64-bit
// row divisions and a conversion an element): the maximum on the bit patterns, and clamp(rint(x 2^e), +-127) as one
// fused multiply-add onto 1.5 2^23, whose low byte is the rounded integer, clamped as a float (NaN gives -127
// there and here).
template <typename InT, int DH>
__device__ __forceinline__ void quant_tokens(int cta, const InT* __restrict__ x, Strides4 xs, int rows, int H,
                                             int8_t* __restrict__ q8, int32_t* __restrict__ eq) {
  constexpr int N = 16 / (int)sizeof(InT), G = DH / N, RPW = 32 / G, RPC = 8 * RPW;
  const int sub = threadIdx.x % G;
  const int row0 = cta * RPC * kRowsPerLane + threadIdx.x / G;
  const bool flat = xs.s1 == H * xs.s2;                  // consecutive rows a head stride apart
  uint4 u[kRowsPerLane];
#pragma unroll
  for (int k = 0; k < kRowsPerLane; ++k) {
    const int row = row0 + k * RPC;
    const int n = flat ? 0 : row / H;
    u[k] = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows) u[k] = __ldg(reinterpret_cast<const uint4*>(x + n * xs.s1 + (row - n * H) * xs.s2 + sub * N));
  }
#pragma unroll
  for (int k = 0; k < kRowsPerLane; ++k) {
    const int row = row0 + k * RPC;
    float m = absmax_value<InT>(absmax_acc<InT>(0u, u[k]));
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int e = pow2_exponent(m, 40);
    const float sc = pow2f(e);
    const InT* xe = reinterpret_cast<const InT*>(&u[k]);
    uint32_t q[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      q[i] = __float_as_uint(fminf(fmaxf(__fmaf_rn(to_f32(xe[i]), sc, 12582912.0f), 12582912.0f - 127.0f), 12582912.0f + 127.0f));
    if (row < rows) {
      int8_t* dst = q8 + (long long)row * DH + sub * N;
      if constexpr (N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(pack4_s8(q[0], q[1], q[2], q[3]), pack4_s8(q[4], q[5], q[6], q[7]));
      else *reinterpret_cast<uint32_t*>(dst) = pack4_s8(q[0], q[1], q[2], q[3]);
      if (sub == 0) eq[row] = e;
    }
  }
}

template <typename Plan, typename InT, int DH>
__global__ void __launch_bounds__(kStepPlanThreads)
step_plan_quant_kernel(const Plan plan, const InT* __restrict__ x, Strides4 xs, int N, int H, int8_t* __restrict__ q8,
                       int32_t* __restrict__ eq) {
  pdl_launch_dependents();                       // the attention kernel may start its setup
  if (blockIdx.x == 0) step_plan(plan);
  else quant_tokens<InT, DH>((int)blockIdx.x - 1, x, xs, N * H, H, q8, eq);
}

}  // namespace lssab8
