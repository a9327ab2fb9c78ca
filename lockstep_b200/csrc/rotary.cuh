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
// Memory-bound: every element is read and written once.  A CTA serves a few tokens: it computes their
// cosines and sines once into shared memory and streams all their heads past them in 16-byte vectors.
#pragma once
#include "common.cuh"

namespace lssab8 {

enum : int { kRotHalf = 0, kRotInterleaved = 1 };            // pairs (i, i + rot/2) / (2i, 2i + 1)
constexpr int kRotThreads = 256;
constexpr int kRotMaxDim = 512;                              // head dim limit (shared memory of a token: 2 KB)

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

// cosine / sine table of ntok tokens (the CTA's) in shared memory: cs[tok * rot / 2 + i]
__device__ __forceinline__ void rot_table(float2* cs, const RotPlan& pl, const RotPos& pos, int b, long long t0,
                                          int ntok) {
  const int np = pl.rot / 2;
  for (int k = threadIdx.x; k < ntok * np; k += blockDim.x) {
    const int tok = k / np, i = k - tok * np;
    cs[k] = turn_cos_sin((unsigned long long)pos.at(b, t0 + tok) * pl.freq[i], pl.factor, pl.sign);
  }
}

__device__ __forceinline__ float rot_lo(float a, float b, float2 cs) { return __fmaf_rn(a, cs.x, -__fmul_rn(b, cs.y)); }
__device__ __forceinline__ float rot_hi(float a, float b, float2 cs) { return __fmaf_rn(b, cs.x, __fmul_rn(a, cs.y)); }

template <typename T, int VEC> struct __align__(sizeof(T) * VEC >= 16 ? 16 : sizeof(T) * VEC) RotVec { T e[VEC]; };

// same type: the value's bits; else one rounding of its binary32 value
template <typename C, typename T> __device__ __forceinline__ C rot_cast(T x) {
  if constexpr (std::is_same<C, T>::value) return x;
  else return from_f32<C>(to_f32(x));
}

// Unit k of one row (one token, one head): the vectors that are read and written together.  Half
// layout: units [0, rot/2/VEC) are a vector of first halves and its partner; the rest, one vector each,
// pass.  Interleaved: one vector, its pairs below rot rotated.  VEC = 1 (any strides and alignment):
// units [0, rot/2) are pairs, the rest single channels.  Both sides of a pair are read before either is
// written, so dst may be src.
template <typename T, typename C, int VEC, int LAYOUT>
__device__ __forceinline__ void rot_unit(const T* src, long long sc, C* dst, long long dc, int k, const RotPlan& pl,
                                         const float2* cs) {
  const int np = pl.rot / 2;
  if constexpr (VEC == 1) {
    if (k < np) {
      const long long c1 = LAYOUT == kRotHalf ? k : 2 * k, c2 = LAYOUT == kRotHalf ? k + np : 2 * k + 1;
      const float a = to_f32(src[c1 * sc]), b = to_f32(src[c2 * sc]);
      dst[c1 * dc] = from_f32<C>(rot_lo(a, b, cs[k]));
      dst[c2 * dc] = from_f32<C>(rot_hi(a, b, cs[k]));
    } else {
      const long long c = k + np;                            // units [np, dh - np): channels [rot, dh)
      dst[c * dc] = rot_cast<C>(src[c * sc]);
    }
  } else if constexpr (LAYOUT == kRotHalf) {
    const int nu = np / VEC;
    if (k < nu) {
      const int c1 = k * VEC, c2 = c1 + np;
      const RotVec<T, VEC> a = *reinterpret_cast<const RotVec<T, VEC>*>(src + c1);
      const RotVec<T, VEC> b = *reinterpret_cast<const RotVec<T, VEC>*>(src + c2);
      RotVec<C, VEC> ya, yb;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float2 w = cs[c1 + i];
        const float x1 = to_f32(a.e[i]), x2 = to_f32(b.e[i]);
        ya.e[i] = from_f32<C>(rot_lo(x1, x2, w));
        yb.e[i] = from_f32<C>(rot_hi(x1, x2, w));
      }
      *reinterpret_cast<RotVec<C, VEC>*>(dst + c1) = ya;
      *reinterpret_cast<RotVec<C, VEC>*>(dst + c2) = yb;
    } else {
      const int c = pl.rot + (k - nu) * VEC;
      const RotVec<T, VEC> a = *reinterpret_cast<const RotVec<T, VEC>*>(src + c);
      RotVec<C, VEC> y;
#pragma unroll
      for (int i = 0; i < VEC; ++i) y.e[i] = rot_cast<C>(a.e[i]);
      *reinterpret_cast<RotVec<C, VEC>*>(dst + c) = y;
    }
  } else {
    const int c = k * VEC;
    const RotVec<T, VEC> a = *reinterpret_cast<const RotVec<T, VEC>*>(src + c);
    RotVec<C, VEC> y;
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const int pr = c / 2 + i / 2;
      if (pr < np) {
        const float2 w = cs[pr];
        const float x1 = to_f32(a.e[i]), x2 = to_f32(a.e[i + 1]);
        y.e[i] = from_f32<C>(rot_lo(x1, x2, w));
        y.e[i + 1] = from_f32<C>(rot_hi(x1, x2, w));
      } else {
        y.e[i] = rot_cast<C>(a.e[i]);
        y.e[i + 1] = rot_cast<C>(a.e[i + 1]);
      }
    }
    *reinterpret_cast<RotVec<C, VEC>*>(dst + c) = y;
  }
}

// units of a row
template <int VEC, int LAYOUT> __host__ __device__ __forceinline__ int rot_units(int rot, int dh) {
  if (VEC == 1) return dh - rot / 2;
  if (LAYOUT == kRotHalf) return rot / 2 / VEC + (dh - rot) / VEC;
  return dh / VEC;
}

// the vector forms' condition on the channel counts (the strides and addresses are checked beside it)
inline bool rot_vec_ok(int vec, int layout, int rot, int dh) {
  if (dh % vec) return false;
  return layout == kRotInterleaved || (rot / 2) % vec == 0;
}

// x [B, H, T, dh] -> y, tokens [t0, t0 + tpc) of batch element b a CTA, heads split over gridDim.y
template <typename T, int VEC, int LAYOUT>
__global__ void __launch_bounds__(kRotThreads)
rotate_kernel(const T* x, long long xb, long long xh, long long xt, long long xc, T* y, long long yb, long long yh,
              long long yt, long long yc, int H, int Tn, int tpc, int hpc, RotPlan pl, RotPos pos) {
  extern __shared__ float2 cs[];
  const int tiles = (Tn + tpc - 1) / tpc;
  const int b = blockIdx.x / tiles;
  const long long t0 = (long long)(blockIdx.x - b * tiles) * tpc;
  const int ntok = (int)min((long long)tpc, Tn - t0);
  rot_table(cs, pl, pos, b, t0, ntok);
  __syncthreads();
  const int h0 = blockIdx.y * hpc, nh = min(hpc, H - h0);
  const int nu = rot_units<VEC, LAYOUT>(pl.rot, pl.dh), np = pl.rot / 2;
  // tokens fastest after the row's units: consecutive rows of one head are adjacent in [B, H, T, dh]
  for (int i = threadIdx.x; i < nh * ntok * nu; i += kRotThreads) {
    const int row = i / nu, k = i - row * nu;
    const int hh = row / ntok, tok = row - hh * ntok;
    rot_unit<T, T, VEC, LAYOUT>(x + b * xb + (h0 + hh) * xh + (t0 + tok) * xt, xc,
                                y + b * yb + (h0 + hh) * yh + (t0 + tok) * yt, yc, k, pl, cs + tok * np);
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

template <typename T, typename C, int VEC, int LAYOUT>
__global__ void __launch_bounds__(kRotThreads)
rotate_append_kernel(const RotAppend a, int tpc, int hpc, RotPlan pl, RotPos pos, int* err) {
  extern __shared__ float2 cs[];
  const long long t0 = (long long)blockIdx.x * tpc;
  const int ntok = (int)min((long long)tpc, a.N - t0);
  rot_table(cs, pl, pos, 0, t0, ntok);
  __syncthreads();
  const int heads = a.H + 2 * a.KVH;
  const int h0 = blockIdx.y * hpc, nh = min(hpc, heads - h0);
  const int nu = rot_units<VEC, LAYOUT>(pl.rot, pl.dh), np = pl.rot / 2;
  for (int i = threadIdx.x; i < nh * ntok * nu; i += kRotThreads) {
    const int row = i / nu, k = i - row * nu;
    const int tok = row / nh, h = h0 + row - tok * nh;       // heads of a token are adjacent
    const long long t = t0 + tok;
    if (h < a.H) {
      rot_unit<T, T, VEC, LAYOUT>(static_cast<const T*>(a.q) + t * a.qt + h * a.qh, 1,
                                  static_cast<T*>(a.qo) + t * a.ot + h * a.oh, 1, k, pl, cs + tok * np);
      continue;
    }
    const long long slot = a.slots[t];
    if (slot < 0 || slot >= a.nslots) {
      if (slot != -1) atomicOr(err, kDevBadPage);
      continue;
    }
    const int g = h - a.H;
    if (g < a.KVH) {
      rot_unit<T, C, VEC, LAYOUT>(static_cast<const T*>(a.k) + t * a.kt + g * a.kh, 1,
                                  static_cast<C*>(a.kc) + (slot >> 4) * a.kp + (slot & 15) * a.kr + g * a.kg, 1, k, pl,
                                  cs + tok * np);
    } else {                                                 // the same units, copied
      const T* src = static_cast<const T*>(a.v) + t * a.vt + (g - a.KVH) * a.vh;
      C* dst = static_cast<C*>(a.vc) + (slot >> 4) * a.vp + (slot & 15) * a.vr + (g - a.KVH) * a.vg;
      if constexpr (VEC == 1) {
        dst[k] = rot_cast<C>(src[k]);
        if (k + nu < pl.dh) dst[k + nu] = rot_cast<C>(src[k + nu]);
      } else {
        for (int c = k * VEC; c < pl.dh; c += nu * VEC) {
          const RotVec<T, VEC> x = *reinterpret_cast<const RotVec<T, VEC>*>(src + c);
          RotVec<C, VEC> y;
#pragma unroll
          for (int e = 0; e < VEC; ++e) y.e[e] = rot_cast<C>(x.e[e]);
          *reinterpret_cast<RotVec<C, VEC>*>(dst + c) = y;
        }
      }
    }
  }
}

}  // namespace lssab8
