// C ABI of the serving-step operators (declarations: include/lssab8.h): rotary positions, step tables,
// packed prompt rows over the paged lattice, and decode over a shared prefix.
#include <atomic>
#include <type_traits>

#include "../../include/lssab8.h"
#include "host.cuh"
#include "rotary.cuh"
#include "tables.cuh"
#include "prefill.cuh"
#include "decode.cuh"
#include "decode_tc.cuh"
#include "paged.cuh"

using namespace lssab8;

namespace {

// A kernel's shared-memory limit, raised once on each device (the runtime call costs 1 us a launch).
struct SmemAttr {
  std::atomic<uint64_t> done{0};
  template <typename K> bool set(K kfn, int smem) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (done.load(std::memory_order_acquire) >> dev & 1) return true;
    if (cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return false;
    done.fetch_or(1ull << dev, std::memory_order_release);
    return true;
  }
};

// ------------------------------------------------------------------ rotary
bool rot_args_ok(const void* freq, int rot, int dh, int layout) {
  return freq && dh > 0 && dh <= kRotMaxDim && rot > 0 && rot <= dh && rot % 2 == 0 &&
         (layout == kRotHalf || layout == kRotInterleaved);
}

// Warps a token: one, or for few tokens as many as give every SM two CTAs, down to four heads a warp.
int rot_chunks(long long tokens, int heads, int sms) {
  const long long want = 2LL * sms * kRotWarps;
  return (int)std::max<long long>(1, std::min<long long>((heads + 3) / 4, want / tokens));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, int VEC>
int launch_rotate(const void* x, const int64_t* xs, void* y, const int64_t* ys, int B, int H, int T_, const RotPlan& pl,
                  const RotPos& pos, int sms, cudaStream_t st) {
  const long long tokens = (long long)B * T_;
  const int chunks = rot_chunks(tokens, H, sms);
  const long long grid = (tokens * chunks + kRotWarps - 1) / kRotWarps;
  if (grid > 0x7FFFFFFF) return kErrArg;
  const bool full = pl.rot == pl.dh && VEC > 1;
  auto kfn = pl.layout == kRotHalf ? (full ? rotate_kernel<T, VEC, kRotHalf, true> : rotate_kernel<T, VEC, kRotHalf, false>)
                                   : (full ? rotate_kernel<T, VEC, kRotInterleaved, true>
                                           : rotate_kernel<T, VEC, kRotInterleaved, false>);
  kfn<<<(unsigned)grid, 32 * kRotWarps, kRotWarps * pl.rot * 4, st>>>(
      static_cast<const T*>(x), xs[0], xs[1], xs[2], xs[3], static_cast<T*>(y), ys[0], ys[1], ys[2], ys[3], B, H, T_, chunks,
      pl, pos);
  return launch_rc();
}

template <typename T, typename C, int VEC>
int launch_append(const RotAppend& a, const RotPlan& pl, const RotPos& pos, const DevState* ds, cudaStream_t st) {
  const int chunks = rot_chunks(a.N, a.H, ds->num_sms), kv_chunks = std::min(chunks, (a.KVH + 3) / 4);
  const long long grid = ((long long)a.N * chunks + kRotWarps - 1) / kRotWarps;
  if (grid > 0x7FFFFFFF) return kErrArg;
  const bool full = pl.rot == pl.dh && VEC > 1;
  auto kfn = pl.layout == kRotHalf ? (full ? rotate_append_kernel<T, C, VEC, kRotHalf, true>
                                           : rotate_append_kernel<T, C, VEC, kRotHalf, false>)
                                   : (full ? rotate_append_kernel<T, C, VEC, kRotInterleaved, true>
                                           : rotate_append_kernel<T, C, VEC, kRotInterleaved, false>);
  kfn<<<dim3((unsigned)grid, 3), 32 * kRotWarps, kRotWarps * pl.rot * 4, st>>>(a, chunks, kv_chunks, pl, pos, ds->err);
  return launch_rc();
}

// ------------------------------------------------------------------ plans
// The call's plan and the quantiser of its queries [N, H, dh] -> q8 [N, H, dh], eq [N, H], in one launch when the
// rows are 16-byte vectors.
template <typename Plan>
int plan_and_quant(const Plan& plan, const void* q, int dtype, int N, int H, int dh, const int64_t* qs, int8_t* q8,
                   int32_t* eq, cudaStream_t st) {
  return with_in_dtype(dtype, [&](auto tag) -> int {
    using InT = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    const Strides4 s{0, qs[0], qs[1], qs[2]};                  // "heads" are tokens, "rows" the token's heads
    if (!vec_ok<InT>(q, s, dh)) {
      step_plan_kernel<Plan><<<1, kStepPlanThreads, 0, st>>>(plan);
      const int rc = launch_rc();
      const int64_t q4[4] = {0, qs[0], qs[1], qs[2]};
      return rc ? rc : lssab8_quant_rows(q, dtype, 1, N, H, dh, q4, H, q8, eq, st);
    }
    const int rpw = 32 / (dh / Vec16<InT>::kN);
    const long long per_cta = 8LL * rpw * kRowsPerLane;
    const long long ctas = ((long long)N * H + per_cta - 1) / per_cta;
    if (dh == 128)
      step_plan_quant_kernel<Plan, InT, 128><<<(unsigned)(ctas + 1), kStepPlanThreads, 0, st>>>(
          plan, static_cast<const InT*>(q), s, N, H, q8, eq);
    else
      step_plan_quant_kernel<Plan, InT, 64><<<(unsigned)(ctas + 1), kStepPlanThreads, 0, st>>>(
          plan, static_cast<const InT*>(q), s, N, H, q8, eq);
    return launch_rc();
  });
}

// q8 [B, H, dh] as boxes of (dh, the kv head's group, sequences): a tile's rows in (sequence, head) order
int make_tmap_group(CUtensorMap* tm, const void* base, int B, int H, int dh, int group, int seqs) {
  const auto encode = encode_fn();
  if (!encode) return kErrCuda;
  cuuint64_t dims[3] = {(cuuint64_t)dh, (cuuint64_t)H, (cuuint64_t)B};
  cuuint64_t strides[2] = {(cuuint64_t)dh, (cuuint64_t)H * dh};
  cuuint32_t box[3] = {(cuuint32_t)dh, (cuuint32_t)group, (cuuint32_t)seqs};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, dh == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? kOk : kErrCuda;
}

// ------------------------------------------------------------------ packed prompt rows
struct RowsWs {
  size_t q8, eq, tile_off, tiles, ntiles, total;
};

RowsWs rows_ws(int N, int H, int dh, int B) {
  RowsWs w{};
  size_t o = 0;
  w.q8 = o; o += align256((size_t)N * H * dh);
  w.eq = o; o += align256((size_t)N * H * 4);
  w.tile_off = o; o += align256((size_t)(B + 1) * 4);
  w.tiles = o; o += align256(((size_t)N / 128 + B) * 16);
  w.ntiles = o; o += 256;
  w.total = o + 256;
  return w;
}

template <int DH, bool SINK, typename OutT, bool MULTI, int SRC>
int launch_paged_t(const CUtensorMap& tq, const CUtensorMap& tk, const PrefillArgs& a, long long items, int num_sms,
                   cudaStream_t st) {
  int smem = kTabBytes + 1024 + PrefillSmem<DH>::kBytes + (SRC == kSrcShared ? 8 * 2048 : 0);   // (the partials' stage)
  if (smem < 116 * 1024) smem = 116 * 1024;                   // one CTA (one 512-column TMEM allocation) an SM
  auto kfn = prefill_kernel<DH, SINK, OutT, MULTI, false, false, SRC>;
  static SmemAttr attr;
  if (!attr.set(kfn, smem)) return kErrCuda;
  const int grid = (int)std::min<long long>(items, (long long)std::max(num_sms, 1));
  return launch_pdl(kfn, dim3(grid), dim3(kPrefillThreads), smem, st, tq, tk, tk, a);
}

template <int DH, bool SINK>
int launch_rows(int out_dtype, bool multi, const CUtensorMap& tq, const CUtensorMap& tk, const PrefillArgs& a,
                long long items, int num_sms, cudaStream_t st) {
  switch (out_dtype) {
    case kF32: return multi ? launch_paged_t<DH, SINK, float, true, kSrcRows>(tq, tk, a, items, num_sms, st)
                            : launch_paged_t<DH, SINK, float, false, kSrcRows>(tq, tk, a, items, num_sms, st);
    case kF16: return multi ? launch_paged_t<DH, SINK, __half, true, kSrcRows>(tq, tk, a, items, num_sms, st)
                            : launch_paged_t<DH, SINK, __half, false, kSrcRows>(tq, tk, a, items, num_sms, st);
    case kBF16: return multi ? launch_paged_t<DH, SINK, __nv_bfloat16, true, kSrcRows>(tq, tk, a, items, num_sms, st)
                             : launch_paged_t<DH, SINK, __nv_bfloat16, false, kSrcRows>(tq, tk, a, items, num_sms, st);
    default: return kErrArg;
  }
}

void prefill_consts(PrefillArgs* a, int dh, int* err) {
  a->gbase = gbase_of(dh);
  a->mul_entry = kTabCopies * 4;
  a->mul_b1 = 1u << 8;
  a->mul_b2 = 1u << 16;
  a->mul_b3 = 1u << 24;
  a->err = err;
  a->wait_ns = kWaitLimitNs;
  a->withhold = -1;
  a->causal = 1;
}

// ------------------------------------------------------------------ shared prefix
// How the shared blocks are cut into items.  Row tiles x kv heads is the work of one block; the items are
// folded segments and, for the rest, chunks of exact partials.
struct SharedShape {
  int seqs_per_tile, row_tiles, nfold, chunk, nchunks;
};
SharedShape shared_shape(int B, int KVH, int group, int shared_blocks, int num_sms) {
  SharedShape s{};
  s.seqs_per_tile = 128 / group;
  s.row_tiles = (B + s.seqs_per_tile - 1) / s.seqs_per_tile;
  const long long per_block = (long long)KVH * s.row_tiles;
  // A folded segment is 32 blocks one after another on one SM (2 us a block); partials run on all SMs at once but
  // cost 6.5 us a block and SM, refold included.  Measured (32 to 128 sequences, groups 4 and 8, prefixes 2,048 to
  // 32,768; partials / folded): 1,024 block tiles 71 / 85 us, 2,048 113 / 87 us, 4,096 186 / 97 us.
  const long long segs = per_block * (shared_blocks / kSEG);
  const long long waves = (segs + num_sms - 1) / num_sms;
  s.nfold = per_block * shared_blocks > waves * kSEG * num_sms * 5 / 16 ? shared_blocks / kSEG : 0;
  const int rest = shared_blocks - s.nfold * kSEG;
  if (rest > 0) {
    const long long slots = std::max<long long>(1, num_sms / per_block);   // items a (tile, kv head) in one wave
    s.chunk = s.nfold ? 4 : (int)((rest + slots - 1) / slots);
    s.nchunks = (rest + s.chunk - 1) / s.chunk;
  }
  return s;
}

struct SharedWs {
  size_t q8, eq, partA, partM, segO, segM, blk_off, order, leader, total;
};
SharedWs shared_ws(int B, int H, int KVH, int dh, int max_part, int nfold) {
  SharedWs w{};
  size_t o = 0;
  w.q8 = o; o += align256((size_t)B * H * dh);
  w.eq = o; o += align256((size_t)B * H * 4);
  w.partA = o; o += align256((size_t)B * H * max_part * dh * 4);
  w.partM = o; o += align256((size_t)B * H * max_part * 16);
  w.segO = o; o += align256((size_t)B * H * nfold * dh * 4);
  w.segM = o; o += align256((size_t)B * H * nfold * 8);
  w.blk_off = o; o += align256((size_t)(B + 1) * 4);
  w.order = o; o += align256((size_t)B * 4);
  w.leader = o; o += 256;
  w.total = o + 256;
  return w;
}

template <bool SINK, typename OutT, int GQ>
int launch_own_tc(const DecodeArgs& a, int num_sms, cudaStream_t st) {
  CUtensorMap tk, tq;
  int rc;
  if ((rc = make_tmap(&tk, a.k8p, (long long)a.num_pages * a.KVH * 16, 128, 16))) return rc;
  if ((rc = make_tmap(&tq, a.q8, (long long)a.B * a.H, 128, 16))) return rc;
  const int smem = DecTcSmem::kBytes + 1024;
  auto kfn = decode_tc_kernel<SINK, OutT, GQ, true>;
  static SmemAttr attr;
  if (!attr.set(kfn, smem)) return kErrCuda;
  const long long blocks = (long long)a.B * a.KVH * (a.max_blocks - a.skip_blocks);
  const int grid = (int)std::max<long long>(1, std::min<long long>(blocks, 2LL * std::max(num_sms, 1)));
  return launch_pdl(kfn, dim3(grid), dim3(DecWorkers<GQ>::kThreads), smem, st, tk, tq, a);
}

template <int DH, bool SINK, typename OutT>
int launch_shared_t(const DecodeArgs& a, const PrefillArgs& pa, const SharedShape& sh, int num_sms, cudaStream_t st) {
  CUtensorMap tk, tq;
  int rc;
  if ((rc = make_tmap(&tk, a.k8p, (long long)a.num_pages * a.KVH * 16, DH, 16))) return rc;
  if ((rc = make_tmap_group(&tq, a.q8, a.B, a.H, DH, a.group, sh.seqs_per_tile))) return rc;
  const long long items = (long long)a.KVH * sh.row_tiles * (sh.nfold + sh.nchunks);
  if ((rc = launch_paged_t<DH, SINK, float, false, kSrcShared>(tq, tk, pa, items, num_sms, st))) return rc;
  if (a.max_blocks > a.skip_blocks) {
    if constexpr (DH == 128) {
      // the output type plays no part before the refold
      rc = a.group == 4 ? launch_own_tc<SINK, float, 4>(a, num_sms, st) : launch_own_tc<SINK, float, 8>(a, num_sms, st);
    } else {
      const int smem = DecodeSmem<DH>::kBytes + 128;
      auto kfn = decode_kernel<DH, SINK, float, true>;
      static SmemAttr attr;
      if (!attr.set(kfn, smem)) return kErrCuda;
      rc = launch_pdl(kfn, dim3((a.max_blocks - a.skip_blocks + a.split_blocks - 1) / a.split_blocks, a.KVH, a.B),
                      dim3(128), smem, st, a);
    }
    if (rc) return rc;
  }
  // (an ordinary launch: its waiting CTAs, started early, cost the kernels before it more than they save; 32 sequences
  // on 8,192 tokens 48.5 -> 45.3 us)
  decode_merge_kernel<SINK, OutT, DH, true><<<dim3(a.group, a.KVH, a.B), kMergeThreads, 0, st>>>(a);
  return launch_rc();
}

template <int DH, bool SINK>
int launch_shared_out(int out_dtype, const DecodeArgs& a, const PrefillArgs& pa, const SharedShape& sh, int num_sms,
                      cudaStream_t st) {
  switch (out_dtype) {
    case kF32: return launch_shared_t<DH, SINK, float>(a, pa, sh, num_sms, st);
    case kF16: return launch_shared_t<DH, SINK, __half>(a, pa, sh, num_sms, st);
    case kBF16: return launch_shared_t<DH, SINK, __nv_bfloat16>(a, pa, sh, num_sms, st);
    default: return kErrArg;
  }
}

int shared_args(int B, int H, int KVH, int dh, int max_blocks, int shared_len, SharedShape* sh, SharedWs* w) {
  if (B <= 0 || B > 65535 || H <= 0 || KVH <= 0 || KVH > 65535 || H % KVH || max_blocks <= 0 || shared_len < kKB ||
      shared_len / kKB > max_blocks)
    return kErrArg;
  if ((dh != 64 && dh != 128) || H / KVH > 8) return kErrUnsupported;
  DevState* ds = nullptr;
  int rc = dev_state(&ds);
  if (rc) return rc;
  *sh = shared_shape(B, KVH, H / KVH, shared_len / kKB, ds->num_sms);
  *w = shared_ws(B, H, KVH, dh, std::max(1, max_blocks - sh->nfold * kSEG), sh->nfold);
  return kOk;
}

}  // namespace

extern "C" {

int lssab8_rotate(const void* x, int dtype, int B, int H, int T, int dh, const int64_t* xs, const void* positions,
                  int pos64, const int64_t* ps, const uint64_t* freq, float factor, int rot, int layout, int inverse,
                  void* y, const int64_t* ys, void* stream) {
  if (!x || !y || !positions || !strides_ok(xs, 4) || !strides_ok(ys, 4) || !strides_ok(ps, 2) || B <= 0 || H <= 0 ||
      T <= 0 || !rot_args_ok(freq, rot, dh, layout))
    return kErrArg;
  DevState* ds = nullptr;
  int rc = dev_state(&ds);
  if (rc) return rc;
  const RotPlan pl{reinterpret_cast<const unsigned long long*>(freq), factor, rot, dh, layout, inverse ? -1.0f : 1.0f};
  const RotPos pos{positions, ps[0], ps[1], pos64};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_in_dtype(dtype, [&](auto tag) -> int {
    using T_ = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    constexpr int VEC = 16 / (int)sizeof(T_);
    bool vec = rot_vec_ok(VEC, layout, rot, dh) && xs[3] == 1 && ys[3] == 1 && aligned16(x) && aligned16(y);
    for (int i = 0; i < 3; ++i) vec = vec && xs[i] % VEC == 0 && ys[i] % VEC == 0;
    return vec ? launch_rotate<T_, VEC>(x, xs, y, ys, B, H, T, pl, pos, ds->num_sms, st)
               : launch_rotate<T_, 1>(x, xs, y, ys, B, H, T, pl, pos, ds->num_sms, st);
  });
}

int lssab8_rotate_append(const void* q, const void* k, const void* v, int dtype, int N, int H, int KVH, int dh,
                         const int64_t* qs, const int64_t* ks, const int64_t* vs, const void* positions, int pos64,
                         int64_t pos_stride, const uint64_t* freq, float factor, int rot, int layout, void* q_out,
                         const int64_t* os, void* k_cache, void* v_cache, int cache_dtype, const int64_t* kcs,
                         const int64_t* vcs, int num_pages, const int64_t* slots, void* stream) {
  if (!q || !k || !v || !q_out || !k_cache || !v_cache || !slots || !positions || !strides_ok(qs, 2) ||
      !strides_ok(ks, 2) || !strides_ok(vs, 2) || !strides_ok(os, 2) || !strides_ok(kcs, 3) || !strides_ok(vcs, 3) ||
      N <= 0 || H <= 0 || KVH <= 0 || num_pages <= 0 || pos_stride < 0 || !rot_args_ok(freq, rot, dh, layout))
    return kErrArg;
  DevState* ds = nullptr;
  int rc = dev_state(&ds);
  if (rc) return rc;
  const RotPlan pl{reinterpret_cast<const unsigned long long*>(freq), factor, rot, dh, layout, 1.0f};
  const RotPos pos{positions, 0, pos_stride, pos64};
  const RotAppend a{q, k, v, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], q_out, os[0], os[1], k_cache, v_cache,
                    kcs[0], kcs[1], kcs[2], vcs[0], vcs[1], vcs[2], reinterpret_cast<const long long*>(slots),
                    16LL * num_pages, N, H, KVH};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_in_dtype(dtype, [&](auto tag) -> int {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    return with_in_dtype(cache_dtype, [&](auto ctag) -> int {
      using C = std::remove_const_t<std::remove_pointer_t<decltype(ctag)>>;
      constexpr int VEC = 16 / (int)sizeof(T);
      constexpr int CV = VEC * (int)sizeof(C) >= 16 ? 16 / (int)sizeof(C) : VEC;    // cache elements an aligned store
      bool vec = rot_vec_ok(VEC, layout, rot, dh) && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) &&
                 aligned16(k_cache) && aligned16(v_cache);
      for (int i = 0; i < 2; ++i)
        vec = vec && qs[i] % VEC == 0 && ks[i] % VEC == 0 && vs[i] % VEC == 0 && os[i] % VEC == 0;
      for (int i = 0; i < 3; ++i) vec = vec && kcs[i] % CV == 0 && vcs[i] % CV == 0;
      return vec ? launch_append<T, C, VEC>(a, pl, pos, ds, st) : launch_append<T, C, 1>(a, pl, pos, ds, st);
    });
  });
}

int lssab8_step_tables(const int32_t* before, const int32_t* fresh, int n, int32_t* block_table, int64_t table_stride,
                       int max_pages, const int32_t* free_pages, int nfree, int cap, int32_t* query_start_loc,
                       int32_t* seq_lens, int64_t* slot_mapping, int64_t* positions, int32_t* seq_index,
                       int32_t* pages_used, void* stream) {
  if (!before || !fresh || !block_table || (nfree > 0 && !free_pages) || !query_start_loc || !seq_lens || !pages_used ||
      (cap > 0 && (!slot_mapping || !positions || !seq_index)) || n <= 0 || max_pages <= 0 || table_stride < max_pages ||
      nfree < 0 || cap < 0)
    return kErrArg;
  if (n > kTblMaxSeqs || cap > kTblMaxTokens) return kErrUnsupported;
  DevState* ds = nullptr;
  int rc = dev_state(&ds);
  if (rc) return rc;
  const TablesArgs a{before, fresh, n, max_pages, nfree, cap, block_table, table_stride, free_pages, query_start_loc,
                     seq_lens, seq_index, pages_used, reinterpret_cast<long long*>(slot_mapping),
                     reinterpret_cast<long long*>(positions), ds->err};
  static SmemAttr attr;                                       // (the most any call needs: calls may run side by side)
  if (!attr.set(step_tables_kernel, (3 * kTblMaxSeqs + 2) * 4)) return kErrCuda;
  const int smem = (3 * n + 2) * 4;
  const int grid = std::max(1, std::min((cap + kTblThreads - 1) / kTblThreads, ds->num_sms));
  step_tables_kernel<<<grid, kTblThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
  return launch_rc();
}

size_t lssab8_prefill_paged_workspace_size(int N, int H, int KVH, int dh, int B) {
  if (B <= 0 || !shape_ok(1, H, KVH, N, dh)) return 0;
  return rows_ws(N, H, dh, B).total;
}

int lssab8_prefill_paged(const void* q, int dtype, const int64_t* qs, int N, int H, int KVH, int dh, const int32_t* cu_q,
                         const int32_t* seq_lens, const int32_t* prefix_lens, const uint8_t* active, int B,
                         const int32_t* block_table, int max_pages, int num_pages, const int8_t* k8p,
                         const int8_t* v8p, const int32_t* ek, const int32_t* ev, const int32_t* ev0, int max_blocks,
                         int sink, void* out, int out_dtype, const int64_t* os, void* workspace, size_t workspace_bytes,
                         void* stream) {
  if (!q || !cu_q || !seq_lens || !block_table || !k8p || !v8p || !ek || !ev || (sink && !ev0) || !out || !workspace ||
      !strides_ok(qs, 3) || !strides_ok(os, 3) || B <= 0 || !shape_ok(1, H, KVH, N, dh) || max_blocks <= 0 ||
      max_pages <= 0 || num_pages <= 0 || (long long)num_pages * KVH * 16 > 0x7FFFFFFFll || !aligned16(k8p) ||
      !aligned16(v8p) ||
      (long long)H * N > 0x7FFFFFFFll || ((long long)N / 128 + B) * H > 0x7FFFFFFFll)
    return kErrArg;
  if (dh != 64 && dh != 128) return kErrUnsupported;
  const RowsWs w = rows_ws(N, H, dh, B);
  if (workspace_bytes < w.total) return kErrWorkspace;
  DevState* ds = nullptr;
  int rc = dev_state(&ds);
  if (rc) return rc;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int8_t* q8 = reinterpret_cast<int8_t*>(base + w.q8);
  int32_t* eq = reinterpret_cast<int32_t*>(base + w.eq);
  int4* tiles = reinterpret_cast<int4*>(base + w.tiles);
  int* ntiles = reinterpret_cast<int*>(base + w.ntiles);
  const RowsPlanArgs pa{cu_q, seq_lens, prefix_lens, active, B, N, max_blocks, max_pages,
                        reinterpret_cast<int*>(base + w.tile_off), tiles, N / 128 + B, ntiles, ds->err};
  if ((rc = plan_and_quant(pa, q, dtype, N, H, dh, qs, q8, eq, st))) return rc;
  CUtensorMap tq, tk;
  if ((rc = make_tmap_group(&tq, q8, N, H, dh, 1, 128))) return rc;
  if ((rc = make_tmap(&tk, k8p, (long long)num_pages * KVH * 16, dh, 16))) return rc;
  PrefillArgs a{};
  a.B = B; a.H = H; a.KVH = KVH; a.T = 0; a.dh = dh; a.Tpad = N; a.group = H / KVH;
  a.eq = eq; a.ek = ek; a.ev = ev; a.ev0 = sink ? ev0 : nullptr;
  a.out = out; a.os1 = os[0]; a.os2 = os[1]; a.os3 = os[2]; a.out_dtype = out_dtype;
  prefill_consts(&a, dh, ds->err);
  a.pg.max_blocks = max_blocks; a.pg.max_pages = max_pages; a.pg.num_pages = num_pages;
  a.pg.block_table = block_table; a.pg.seq_lens = seq_lens; a.pg.v8p = v8p;
  a.pg.tiles = tiles; a.pg.ntiles = ntiles; a.pg.prefix = prefix_lens;
  const long long items = ((long long)N / 128 + B) * H;       // at most: the plan knows how many
  const bool multi = max_blocks > kSEG;
  if (dh == 128) return sink ? launch_rows<128, true>(out_dtype, multi, tq, tk, a, items, ds->num_sms, st)
                             : launch_rows<128, false>(out_dtype, multi, tq, tk, a, items, ds->num_sms, st);
  return sink ? launch_rows<64, true>(out_dtype, multi, tq, tk, a, items, ds->num_sms, st)
              : launch_rows<64, false>(out_dtype, multi, tq, tk, a, items, ds->num_sms, st);
}

size_t lssab8_decode_shared_workspace_size(int B, int H, int KVH, int dh, int max_blocks, int shared_len) {
  SharedShape sh;
  SharedWs w;
  return shared_args(B, H, KVH, dh, max_blocks, shared_len, &sh, &w) == kOk ? w.total : 0;
}

int lssab8_decode_shared(const void* q, int dtype, const int64_t* qs, int B, int H, int KVH, int dh,
                         const int32_t* seq_lens, int shared_len, const int32_t* block_table, int max_pages,
                         int num_pages, const int8_t* k8p, const int8_t* v8p, const int32_t* ek, const int32_t* ev,
                         const int32_t* ev0, int max_blocks, int sink, void* out, int out_dtype, const int64_t* os,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !seq_lens || !block_table || !k8p || !v8p || !ek || !ev || (sink && !ev0) || !out || !workspace ||
      !strides_ok(qs, 3) || !strides_ok(os, 3) || max_pages <= 0 || num_pages <= 0 ||
      (long long)num_pages * KVH * 16 > 0x7FFFFFFFll || !aligned16(k8p) || !aligned16(v8p))
    return kErrArg;
  SharedShape sh;
  SharedWs w;
  int rc = shared_args(B, H, KVH, dh, max_blocks, shared_len, &sh, &w);
  if (rc) return rc;
  const int shared_blocks = shared_len / kKB;
  if (max_pages < shared_blocks * 8) return kErrArg;
  if (workspace_bytes < w.total) return kErrWorkspace;
  DevState* ds = nullptr;
  if ((rc = dev_state(&ds))) return rc;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int8_t* q8 = reinterpret_cast<int8_t*>(base + w.q8);
  int32_t* eq = reinterpret_cast<int32_t*>(base + w.eq);
  int* leader = reinterpret_cast<int*>(base + w.leader);
  DecodeArgs a{};
  a.B = B; a.H = H; a.KVH = KVH; a.dh = dh; a.group = H / KVH; a.max_blocks = max_blocks; a.max_pages = max_pages;
  a.split_blocks = 4; a.num_pages = num_pages; a.seq_lens = seq_lens; a.block_table = block_table;
  a.k8p = k8p; a.v8p = v8p; a.ek = ek; a.ev = ev; a.ev0 = sink ? ev0 : nullptr; a.q8 = q8; a.eq = eq;
  a.partA = reinterpret_cast<int32_t*>(base + w.partA);
  a.partM = reinterpret_cast<int4*>(base + w.partM);
  a.blk_off = reinterpret_cast<int*>(base + w.blk_off);
  a.order = reinterpret_cast<int*>(base + w.order);
  a.out = out; a.os0 = os[0]; a.os1 = os[1]; a.os2 = os[2];
  a.gbase = gbase_of(dh);
  a.err = ds->err;
  a.skip_blocks = shared_blocks; a.nfold = sh.nfold; a.max_part = std::max(1, max_blocks - sh.nfold * kSEG);
  a.leader = leader;
  a.segO = reinterpret_cast<float*>(base + w.segO);
  a.segM = reinterpret_cast<int2*>(base + w.segM);
  PrefillArgs p{};
  p.B = B; p.H = H; p.KVH = KVH; p.dh = dh; p.group = a.group; p.eq = eq; p.ek = ek; p.ev = ev; p.ev0 = a.ev0;
  prefill_consts(&p, dh, ds->err);
  p.pg.max_blocks = max_blocks; p.pg.max_pages = max_pages; p.pg.num_pages = num_pages;
  p.pg.block_table = block_table; p.pg.seq_lens = seq_lens; p.pg.v8p = v8p;
  p.pg.leader = leader; p.pg.seqs_per_tile = sh.seqs_per_tile; p.pg.row_tiles = sh.row_tiles;
  p.pg.nfold = sh.nfold; p.pg.chunk = sh.chunk; p.pg.nchunks = sh.nchunks; p.pg.shared_blocks = shared_blocks;
  p.pg.max_part = a.max_part; p.pg.partA = a.partA; p.pg.partM = a.partM;
  p.pg.segO = reinterpret_cast<float*>(base + w.segO);
  p.pg.segM = reinterpret_cast<int2*>(base + w.segM);
  const SharedPlanArgs plan{seq_lens, B, max_blocks, max_pages, a.blk_off, a.order, ds->err, shared_blocks, leader};
  if ((rc = plan_and_quant(plan, q, dtype, B, H, dh, qs, q8, eq, st))) return rc;
  if (dh == 128) return sink ? launch_shared_out<128, true>(out_dtype, a, p, sh, ds->num_sms, st)
                             : launch_shared_out<128, false>(out_dtype, a, p, sh, ds->num_sms, st);
  return sink ? launch_shared_out<64, true>(out_dtype, a, p, sh, ds->num_sms, st)
              : launch_shared_out<64, false>(out_dtype, a, p, sh, ds->num_sms, st);
}

}  // extern "C"
