// Host helpers shared by the library's translation units: the per-device state (error word, SM count),
// TMA tensor-map encoding, dtype dispatch, launches with programmatic dependent launch, and the argument
// checks every entry point makes.  dev_state and encode_fn are defined once, in capi.cu.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <utility>

#include "common.cuh"
#include "prep.cuh"

namespace lssab8 {

struct DevState {
  int* err = nullptr;
  bool prefill_attr_set = false;
  int num_sms = 0;
};
// The current device's state.
__attribute__((visibility("hidden"))) int dev_state(DevState** out);
// cuTensorMapEncodeTiled, looked up in the driver once (null: not found).
__attribute__((visibility("hidden"))) PFN_cuTensorMapEncodeTiled_v12000 encode_fn();
// rows x dh int8 matrix, box 128 rows x dh, swizzle = dh bytes
// 2-D int8 tensor map over [rows, dh] (row pitch dh bytes), boxes of box_rows x dh, swizzled for
// the UMMA K-major layouts (128B swizzle at dh 128, 64B at dh 64).
inline int make_tmap(CUtensorMap* tm, const void* base, long long rows, int dh, int box_rows = 128) {
  const auto encode = encode_fn();
  if (!encode) return kErrCuda;
  if ((reinterpret_cast<uintptr_t>(base) & 15) != 0) return kErrArg;
  cuuint64_t dims[2] = {(cuuint64_t)dh, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)dh};
  cuuint32_t box[2] = {(cuuint32_t)dh, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE,
                        dh == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? kOk : kErrCuda;
}

inline int cuda_rc(cudaError_t e) { return e == cudaSuccess ? kOk : kErrCuda; }
inline int launch_rc() { return cuda_rc(cudaGetLastError()); }

inline uint32_t gbase_of(int dh) {
  // round(2^26 / (sqrt(dh) ln 2)) with round-half-even, as Python's round() on the double
  // (reference/lssab_golden.py:161).
  double x = std::ldexp(1.0, kBHI) / (std::sqrt((double)dh) * std::log(2.0));
  return (uint32_t)std::nearbyint(x);
}

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
inline int tpad_of(int T) { return ((T + 127) / 128) * 128; }

// ------------------------------------------------------------------ kernel dispatch helpers
template <typename F>
int with_in_dtype(int dtype, F&& f) {
  switch (dtype) {
    case kF32: return f((const float*)nullptr);
    case kF16: return f((const __half*)nullptr);
    case kBF16: return f((const __nv_bfloat16*)nullptr);
    default: return kErrArg;
  }
}

// Launch with programmatic dependent launch: the kernel may start while the previous kernel on
// the stream finishes; it executes griddepcontrol.wait before it reads that kernel's output.
template <typename... KArgs, typename... Args>
int launch_pdl(void (*kfn)(KArgs...), dim3 grid, dim3 block, int smem, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_rc(cudaLaunchKernelEx(&cfg, kfn, std::forward<Args>(args)...));
}

// the vectorised quantisers need a contiguous channel dim, dh in {64, 128} and 16-byte aligned
// rows (base and every stride a multiple of 16 bytes)
template <typename InT>
bool vec_ok(const void* x, const Strides4& s, int dh) {
  const long long e = (long long)sizeof(InT);
  return (dh == 64 || dh == 128) && s.s3 == 1 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
         (s.s0 * e) % 16 == 0 && (s.s1 * e) % 16 == 0 && (s.s2 * e) % 16 == 0;
}

inline bool strides_ok(const int64_t* s, int n) {
  if (!s) return false;
  for (int i = 0; i < n; ++i) if (s[i] < 0) return false;
  return true;
}

inline bool shape_ok(int B, int H, int KVH, int T, int dh) {
  return B > 0 && H > 0 && KVH > 0 && T > 0 && dh > 0 && H % KVH == 0 && dh <= 256 && dh % 32 == 0 &&
         (long long)T <= (1ll << 24);
}

}  // namespace lssab8
