// Rotary positions: pairs of channels rotated by an angle proportional to the token's position.
//
// Pair i (of rot / 2) of a token at position p turns by p theta_i.  The caller gives theta_i as a
// fraction of a turn in 64-bit fixed point, F_i = theta_i / (2 pi) 2^64, so p F_i mod 2^64 is the
// angle's fraction of a turn exactly: an integer product loses nothing at far positions, where a
// binary32 angle p theta has no fraction left.  The fraction is cut to within an eighth of a turn of
// a quarter turn (exact), rounded once to binary32 and given to sincospif; the quarter turns are
// swaps and signs.  Rotation:  y1 = m (x1 cos - x2 sin),  y2 = m (x2 cos + x1 sin), in binary32 with
// one fused step each, rounded once to the output type.  The inverse (the transposed map, which is the
// gradient) negates the sine.
//
// Memory-bound: every element is read and written once, so what counts is few instructions an element and
// loads in flight.  A warp takes a token: it computes the token's cosines and sines once (rot / 2 of them, exchanged
// through its own shared memory), each lane keeps those of its unit of a row in registers, and the warp then
// streams the token's heads past them, 32 / units rows at a time, 64 bytes a lane in flight, the addresses a fixed
// step apart.  Few tokens: a token's heads are split over several warps.  Measured on a B200 (6.44 TB/s copy): 16,384
// tokens of 64 + 8 + 8 bf16 heads with the cache store 111 us (6.0 TB/s), float32 into a bf16 cache 193 us (6.6); a
// 4 x 32 x 2047 x 128 rotation 45 us float32 (5.9), 28 us bf16.  64 tokens of 32 + 4 + 4 heads: 2.8 us, a launch.
// (With the coefficients read from shared memory for every row the bf16 store took 154 us.)
#pragma once
#include <type_traits>

#include "common.cuh"

namespace lssab8 {

enum : int { kRotHalf = 0, kRotInterleaved = 1 };            // pairs (i, i + rot/2) / (2i, 2i + 1)
constexpr int kRotWarps = 8;
constexpr int kRotMaxDim = 512;                              // head dim limit (a warp's table: at most 2 KB)

struct RotPlan {
  const unsigned long long* freq;     // [rot / 2] turns a position, 2^64 = one turn
  float factor;                       // m
  int rot, dh, layout;
  float sign;                         // +1, or -1 for the inverse
};

// positions of [B, T] tokens: int32 or int64, any strides (0: shared by the batch)
struct RotPos {
  const void* p;
  long long sb, st;
  int is64;
  __device__ __forceinline__ long long at(int b, long long t) const {
    const long long i = b * sb + t * st;
    return is64 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
  }
};

// m (cos, sign sin) of u / 2^64 turns
__device__ __forceinline__ float2 turn_cos_sin(unsigned long long u, float m, float sign) {
  const unsigned long long n = (u + (1ull << 61)) >> 62;     // nearest quarter turn (0 .. 3)
  const long long r = (long long)(u - (n << 62));            // |r| <= 2^61
  float s, c;
  sincospif(__fmul_rn(__ll2float_rn(r), 0x1p-63f), &s, &c);
  const float cc = (n & 1) ? s : c, ss = (n & 1) ? c : s;
  const float cq = (n == 1 || n == 2) ? -cc : cc;
  const float sq = (n >= 2) ? -ss : ss;
  return make_float2(__fmul_rn(cq, m), __fmul_rn(__fmul_rn(sq, m), sign));
}

__device__ __forceinline__ float rot_lo(float a, float b, float2 cs) { return __fmaf_rn(a, cs.x, -__fmul_rn(b, cs.y)); }
__device__ __forceinline__ float rot_hi(float a, float b, float2 cs) { return __fmaf_rn(b, cs.x, __fmul_rn(a, cs.y)); }

template <typename T, int VEC> struct __align__(sizeof(T) * VEC >= 16 ? 16 : sizeof(T) * VEC) RotVec { T e[VEC]; };

// same type: the value's bits; else one rounding of its binary32 value
template <typename C, typename T> __device__ __forceinline__ C rot_cast(T x) {
  if constexpr (std::is_same<C, T>::value) return x;
  else return from_f32<C>(to_f32(x));
}

// A row (one token, one head) is cut into units: the vectors that a lane reads and writes together.
//   half layout      a vector of first halves and its partner; then two vectors each of the passed channels
//   interleaved      one vector, its pairs below rot rotated
// VEC = 1 (any strides and alignment): a pair of channels, then single passed channels.  A unit's two sides are read
// before either is written, so y may be x; a unit without a second side has the first one twice.
struct RotUnit { int o1, o2, pair; };                        // channels, the first pair (< 0: passed)
template <int VEC, int LAYOUT>
__device__ __forceinline__ RotUnit rot_unit(const RotPlan& pl, int k) {
  const int np = pl.rot / 2;
  if constexpr (VEC == 1) {
    if (k >= np) return {k + np, k + np, -1};                // units [np, dh - np): channels [rot, dh)
    return LAYOUT == kRotHalf ? RotUnit{k, k + np, k} : RotUnit{2 * k, 2 * k + 1, k};
  } else if constexpr (LAYOUT == kRotHalf) {
    const int c = k * VEC;
    if (c < np) return {c, c + np, c};
    const int first = pl.rot + (c - np), second = first + ((pl.dh - pl.rot) / VEC + 1) / 2 * VEC;
    return {first, second < pl.dh ? second : first, -1};
  } else {
    return {k * VEC, k * VEC, k * VEC < pl.rot ? k * VEC / 2 : -1};
  }
}
// units of a row
template <int VEC, int LAYOUT> __host__ __device__ __forceinline__ int rot_units(int rot, int dh) {
  if (VEC == 1) return dh - rot / 2;
  if (LAYOUT == kRotHalf) return rot / 2 / VEC + ((dh - rot) / VEC + 1) / 2;
  return dh / VEC;
}

// the vector forms' condition on the channel counts (the strides and addresses are checked beside it)
inline bool rot_vec_ok(int vec, int layout, int rot, int dh) {
  if (dh % vec) return false;
  return layout == kRotInterleaved || (rot / 2) % vec == 0;
}

template <int VEC, int LAYOUT> struct RotForm {
  static constexpr bool kTwo = VEC == 1 || LAYOUT == kRotHalf;              // units of two sides
  static constexpr int kPairs = VEC == 1 ? 1 : LAYOUT == kRotHalf ? VEC : VEC / 2;
};
template <typename T, int VEC> struct RotRegs { RotVec<T, VEC> a, b; };
template <typename T, int VEC, int LAYOUT>
__device__ __forceinline__ void rot_load(RotRegs<T, VEC>& r, const T* src, long long sc, const RotUnit& u) {
  r.a = *reinterpret_cast<const RotVec<T, VEC>*>(src + u.o1 * sc);
  if (RotForm<VEC, LAYOUT>::kTwo) r.b = *reinterpret_cast<const RotVec<T, VEC>*>(src + u.o2 * sc);
}
// two values of a row in one rounding instruction
__device__ __forceinline__ void rot_pack2(float* e, float a, float b) { e[0] = a; e[1] = b; }
__device__ __forceinline__ void rot_pack2(__half* e, float a, float b) {
  *reinterpret_cast<__half2*>(e) = __floats2half2_rn(a, b);
}
__device__ __forceinline__ void rot_pack2(__nv_bfloat16* e, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(e) = __floats2bfloat162_rn(a, b);
}
// A lane's unit: where it lies in a row, and the coefficients of its pairs.  FULL: every channel is rotated.
template <int VEC, int LAYOUT> struct RotLane {
  static constexpr int kPairs = RotForm<VEC, LAYOUT>::kPairs;
  RotUnit u;
  int np;
  float2 w[kPairs];
  __device__ __forceinline__ void load(const RotPlan& pl, const float2* cs, int k) {
    u = rot_unit<VEC, LAYOUT>(pl, k);
    np = pl.rot / 2;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) w[i] = cs[u.pair < 0 ? 0 : min(u.pair + i, np - 1)];
  }
};
template <typename T, typename C, int VEC, int LAYOUT, bool FULL>
__device__ __forceinline__ void rot_store(const RotRegs<T, VEC>& r, C* dst, long long dc, const RotLane<VEC, LAYOUT>& ln) {
  const RotUnit& u = ln.u;
  RotVec<C, VEC> ya, yb;
  if constexpr (VEC == 1) {
    const float x1 = to_f32(r.a.e[0]), x2 = to_f32(r.b.e[0]);
    ya.e[0] = from_f32<C>(rot_lo(x1, x2, ln.w[0]));
    yb.e[0] = from_f32<C>(rot_hi(x1, x2, ln.w[0]));
  } else if constexpr (LAYOUT == kRotHalf) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float a0 = to_f32(r.a.e[i]), b0 = to_f32(r.b.e[i]), a1 = to_f32(r.a.e[i + 1]), b1 = to_f32(r.b.e[i + 1]);
      rot_pack2(&ya.e[i], rot_lo(a0, b0, ln.w[i]), rot_lo(a1, b1, ln.w[i + 1]));
      rot_pack2(&yb.e[i], rot_hi(a0, b0, ln.w[i]), rot_hi(a1, b1, ln.w[i + 1]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float a0 = to_f32(r.a.e[i]), b0 = to_f32(r.a.e[i + 1]);
      rot_pack2(&ya.e[i], rot_lo(a0, b0, ln.w[i / 2]), rot_hi(a0, b0, ln.w[i / 2]));
      if (!FULL && u.pair + i / 2 >= ln.np) {                // the vector in which the rotated part ends
        ya.e[i] = rot_cast<C>(r.a.e[i]);
        ya.e[i + 1] = rot_cast<C>(r.a.e[i + 1]);
      }
    }
  }
  if (!FULL && u.pair < 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      ya.e[i] = rot_cast<C>(r.a.e[i]);
      if (RotForm<VEC, LAYOUT>::kTwo) yb.e[i] = rot_cast<C>(r.b.e[i]);
    }
  }
  *reinterpret_cast<RotVec<C, VEC>*>(dst + u.o1 * dc) = ya;
  if (RotForm<VEC, LAYOUT>::kTwo) *reinterpret_cast<RotVec<C, VEC>*>(dst + u.o2 * dc) = yb;
}
template <typename T, typename C, int VEC, int LAYOUT>
__device__ __forceinline__ void copy_store(const RotRegs<T, VEC>& r, C* dst, const RotUnit& u) {
  RotVec<C, VEC> y;
#pragma unroll
  for (int i = 0; i < VEC; ++i) y.e[i] = rot_cast<C>(r.a.e[i]);
  *reinterpret_cast<RotVec<C, VEC>*>(dst + u.o1) = y;
  if (RotForm<VEC, LAYOUT>::kTwo) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) y.e[i] = rot_cast<C>(r.b.e[i]);
    *reinterpret_cast<RotVec<C, VEC>*>(dst + u.o2) = y;
  }
}

// Heads h of a token, first, first + step, ... below end, through this lane's unit: several rows' loads are issued
// before the first is used (64 bytes a lane; more costs registers and with them resident warps).
template <typename T, typename C, int VEC, int LAYOUT, typename Store>
__device__ __forceinline__ void rot_heads(const T* src, long long sh, long long sc, C* dst, long long dh, int first,
                                          int end, int step, const RotUnit& u, Store store) {
  constexpr int kBytes = VEC * (int)sizeof(T) * (RotForm<VEC, LAYOUT>::kTwo ? 2 : 1);
  constexpr int kUnroll = kBytes >= 32 ? 2 : 4;
  src += first * sh;
  dst += first * dh;
  const long long ss = step * sh, ds = step * dh;
  int h = first;
#pragma unroll 1
  for (; h + (kUnroll - 1) * step < end; h += kUnroll * step) {
    RotRegs<T, VEC> r[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) rot_load<T, VEC, LAYOUT>(r[j], src + j * ss, sc, u);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) store(r[j], dst + j * ds);
    src += kUnroll * ss;
    dst += kUnroll * ds;
  }
#pragma unroll 1
  for (; h < end; h += step) {
    RotRegs<T, VEC> r;
    rot_load<T, VEC, LAYOUT>(r, src, sc, u);
    store(r, dst);
    src += ss;
    dst += ds;
  }
}

// This warp's task: heads [h0, h1) of token n; its table in shared memory.
struct RotTask { long long n; int h0, h1; float2* cs; };
__device__ __forceinline__ bool rot_task(RotTask& t, long long tokens, int heads, int chunks, float2* smem, int np) {
  const long long task = (long long)blockIdx.x * kRotWarps + (threadIdx.x >> 5);
  t.n = chunks == 1 ? task : task / chunks;
  if (t.n >= tokens) return false;
  const int c = chunks == 1 ? 0 : (int)(task - t.n * chunks), hpc = (heads + chunks - 1) / chunks;
  t.h0 = c * hpc;
  t.h1 = min(t.h0 + hpc, heads);
  t.cs = smem + (threadIdx.x >> 5) * np;
  return true;
}
__device__ __forceinline__ void rot_table(float2* cs, const RotPlan& pl, long long position) {
  for (int i = threadIdx.x & 31; i < pl.rot / 2; i += 32)
    cs[i] = turn_cos_sin((unsigned long long)position * pl.freq[i], pl.factor, pl.sign);
  __syncwarp();
}
// The lanes' places in 32 / units rows (one row of 32 units at a time when a row has more)
#define ROT_FOR_LANE_UNITS(VEC, LAYOUT)                                                       \
  const int nu = rot_units<VEC, LAYOUT>(pl.rot, pl.dh), lane = threadIdx.x & 31;              \
  const int rows = nu < 32 ? 32 / nu : 1, r0 = nu < 32 ? lane / nu : 0;                       \
  for (int k = nu < 32 ? lane - r0 * nu : lane; k < nu && r0 < rows; k += nu < 32 ? nu : 32)

// x [B, H, T, dh] -> y
template <typename T, int VEC, int LAYOUT, bool FULL>
__global__ void __launch_bounds__(32 * kRotWarps)
rotate_kernel(const T* x, long long xb, long long xh, long long xt, long long xc, T* y, long long yb, long long yh,
              long long yt, long long yc, int B, int H, int Tn, int chunks, RotPlan pl, RotPos pos) {
  extern __shared__ float2 smem[];
  RotTask t;
  if (!rot_task(t, (long long)B * Tn, H, chunks, smem, pl.rot / 2)) return;
  const int b = (int)(t.n / Tn);
  const long long tok = t.n - (long long)b * Tn;
  rot_table(t.cs, pl, pos.at(b, tok));
  x += b * xb + tok * xt;
  y += b * yb + tok * yt;
  ROT_FOR_LANE_UNITS(VEC, LAYOUT) {
    RotLane<VEC, LAYOUT> ln;
    ln.load(pl, t.cs, k);
    rot_heads<T, T, VEC, LAYOUT>(x, xh, xc, y, yh, t.h0 + r0, t.h1, rows, ln.u,
                         [&](const RotRegs<T, VEC>& r, T* d) { rot_store<T, T, VEC, LAYOUT, FULL>(r, d, yc, ln); });
  }
}

// One step's tokens: q [N, H, dh] rotated into qo, k [N, KVH, dh] rotated and v [N, KVH, dh] copied into
// the paged float cache (16-token pages) at slot page * 16 + row; slot -1 stores nothing.
struct RotAppend {
  const void *q, *k, *v;
  long long qt, qh, kt, kh, vt, vh;          // token and head strides
  void* qo;
  long long ot, oh;
  void *kc, *vc;
  long long kp, kr, kg, vp, vr, vg;          // page, row and head strides of the caches
  const long long* slots;
  long long nslots;                          // 16 * pages
  int N, H, KVH;
};

template <typename T, typename C, int VEC, int LAYOUT, bool FULL>
__global__ void __launch_bounds__(32 * kRotWarps)
rotate_append_kernel(const RotAppend a, int chunks, int kv_chunks, RotPlan pl, RotPos pos, int* err) {
  extern __shared__ float2 smem[];
  RotTask t;
  // CTA rows 0, 1, 2: queries, keys, values (one kind a warp keeps its registers few)
  const int kind = blockIdx.y;
  if (!rot_task(t, a.N, kind == 0 ? a.H : a.KVH, kind == 0 ? chunks : kv_chunks, smem, pl.rot / 2)) return;
  if (kind == 0) {
    rot_table(t.cs, pl, pos.at(0, t.n));
    ROT_FOR_LANE_UNITS(VEC, LAYOUT) {
      RotLane<VEC, LAYOUT> ln;
      ln.load(pl, t.cs, k);
      rot_heads<T, T, VEC, LAYOUT>(static_cast<const T*>(a.q) + t.n * a.qt, a.qh, 1, static_cast<T*>(a.qo) + t.n * a.ot, a.oh,
                           t.h0 + r0, t.h1, rows, ln.u,
                           [&](const RotRegs<T, VEC>& r, T* d) { rot_store<T, T, VEC, LAYOUT, FULL>(r, d, 1, ln); });
    }
    return;
  }
  const long long slot = a.slots[t.n], page = slot >> 4, row = slot & 15;
  if (slot < 0 || slot >= a.nslots) {
    if (slot != -1 && (threadIdx.x & 31) == 0) atomicOr(err, kDevBadPage);
    return;
  }
  if (kind == 1) {
    rot_table(t.cs, pl, pos.at(0, t.n));
    ROT_FOR_LANE_UNITS(VEC, LAYOUT) {
      RotLane<VEC, LAYOUT> ln;
      ln.load(pl, t.cs, k);
      rot_heads<T, C, VEC, LAYOUT>(static_cast<const T*>(a.k) + t.n * a.kt, a.kh, 1,
                           static_cast<C*>(a.kc) + page * a.kp + row * a.kr, a.kg, t.h0 + r0, t.h1, rows, ln.u,
                           [&](const RotRegs<T, VEC>& r, C* d) { rot_store<T, C, VEC, LAYOUT, FULL>(r, d, 1, ln); });
    }
    return;
  }
  ROT_FOR_LANE_UNITS(VEC, LAYOUT) {
    const RotUnit u = rot_unit<VEC, LAYOUT>(pl, k);           // the same units, copied
    rot_heads<T, C, VEC, LAYOUT>(static_cast<const T*>(a.v) + t.n * a.vt, a.vh, 1,
                         static_cast<C*>(a.vc) + page * a.vp + row * a.vr, a.vg, t.h0 + r0, t.h1, rows, u,
                         [&](const RotRegs<T, VEC>& r, C* d) { copy_store<T, C, VEC, LAYOUT>(r, d, u); });
  }
}

}  // namespace lssab8
