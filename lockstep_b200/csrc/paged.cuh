// Attention over the paged lattice for whole steps: the plan of the packed prompt rows, and the launch that
// plans a call and quantises its queries.  (Their kernel,
// and the shared-prefix kernel, are prefill_kernel's paged forms, prefill.cuh; a shared batch's own
// blocks and refold are the decode kernels' SHARED forms.)
#pragma once
#include <type_traits>

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
        if (blocks_of(L) > p.max_blocks || pages_of(L) > p.max_pages) atomicOr(p.err, kDevBadPage);
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
    if (kt * kKB < P) nb = max(nb, blocks_of(P));
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
  step_plan(plan);
}
// max |x| over a 16-byte vector as a bit pattern, NaN included (a pattern above infinity's)
template <typename InT> __device__ __forceinline__ uint32_t absbits(const uint4& v) {
  if constexpr (sizeof(InT) == 2) {
    const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
    return max(m & 0xFFFFu, m >> 16);
  } else {
    return max(max(v.x & 0x7FFFFFFFu, v.y & 0x7FFFFFFFu), max(v.z & 0x7FFFFFFFu, v.w & 0x7FFFFFFFu));
  }
}
// P1 over tokens [N, H, dh] (strides 0, token, head; contiguous channels, 16-byte rows): row n H + h of q8 and eq.
// quant_rows_vec's rule in fewer instructions, which bound it on these rows (16,700 tokens of 32 bf16 heads: 67 us with
// its 64-bit row divisions and a conversion an element, 36 us so, 5.7 TB/s): the maximum on the bit patterns, and rint(x 2^e) as
// one fused multiply-add onto 1.5 2^23, whose low byte is the rounded integer.  |x| 2^e <= 127 by the choice of e,
// except in a row whose exponent was clamped (e = -32) or that holds a NaN: such a row takes the clamped form, its
// maximum without the NaN, and NaN gives -127, as there.
template <typename InT, int DH>
__device__ __forceinline__ void quant_tokens(int cta, const InT* __restrict__ x, Strides4 xs, int rows, int H,
                                             int8_t* __restrict__ q8, int32_t* __restrict__ eq) {
  constexpr int N = 16 / (int)sizeof(InT), G = DH / N, RPW = 32 / G, RPC = 8 * RPW;
  constexpr uint32_t kInf = std::is_same<InT, float>::value ? 0x7F800000u : std::is_same<InT, __half>::value ? 0x7C00u : 0x7F80u;
  constexpr float kMagic = 12582912.0f;                  // 1.5 2^23
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
    uint32_t bits = absbits<InT>(u[k]);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    float m;
    if constexpr (std::is_same<InT, float>::value) m = __uint_as_float(bits);
    else if constexpr (std::is_same<InT, __half>::value) m = __half2float(__ushort_as_half((unsigned short)bits));
    else m = __uint_as_float(bits << 16);
    int e = pow2_exponent(m, 40);
    const bool clamp = bits > kInf || e == -32;
    if (__any_sync(0xffffffffu, clamp)) {                // rare: the maximum without NaN
      m = absmax_value<InT>(absmax_acc<InT>(0u, u[k]));
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      e = pow2_exponent(m, 40);
    }
    const float sc = pow2f(e);
    const InT* xe = reinterpret_cast<const InT*>(&u[k]);
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = __fmaf_rn(to_f32(xe[i]), sc, kMagic);
    if (clamp) {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = fminf(fmaxf(y[i], kMagic - 127.0f), kMagic + 127.0f);
    }
    uint32_t q[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      q[i] = pack4_s8(__float_as_int(y[4 * i]), __float_as_int(y[4 * i + 1]), __float_as_int(y[4 * i + 2]),
                      __float_as_int(y[4 * i + 3]));
    if (row < rows) {
      int8_t* dst = q8 + (long long)row * DH + sub * N;
      if constexpr (N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(q[0], q[1]);
      else *reinterpret_cast<uint32_t*>(dst) = q[0];
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
