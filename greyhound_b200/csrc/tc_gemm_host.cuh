// Host side of the tcgen05 GEMM: tensor maps, tile choice and launches, shared
// by the linear cross-entropy and the linear log-probability pipelines.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdio>
#include <cstdlib>
#include <mutex>

#include "tc_gemm.cuh"

namespace gh {

// One GEMM operand: pointer, pitch, majorness.
struct Operand {
  const void* ptr;
  int64_t ld;
  int mn_major;  // 0: [rows, K] K contiguous; 1: [K, rows] rows contiguous
  // > 0 (A): only this much of K is there; K = 2 * wrap rounded up to 64 takes it
  // twice, each time with zeros up to the round number
  int64_t wrap = 0;
};

// L2 policies of one GEMM: operand loads (0 none, 1 evict_first, 2 evict_last)
// and evict-first output stores.
struct Hints {
  int a = 0, b = 0, out = 0;
};
// Output rows split into bands stored on the ranks that reduce them
// (gemm::Params::peer_out).
struct PeerOut {
  int n = 0;
  int64_t rows = 0;
  int first = 0;  // band whose tiles this GEMM computes first
  void* ptr[gemm::kMaxPeers] = {};
};

// D[M,N] = scale * A B^T (+ addend), D written as out_dtype with pitch ldo
// (defined in lce.cu).
int run_gemm(int dtype, const Operand& A, const Operand& B, int64_t M, int64_t N, int64_t K, void* out,
             int out_dtype, int64_t ldo, const float* add_f32, const void* add_same, int64_t ldadd,
             const float* scale, int raster, int max_ctas, cudaStream_t st, int* status,
             int prof_class = PROF_GEMM_OTHER, Hints hints = Hints{}, void* split_out = nullptr,
             const float* row_scale = nullptr, const PeerOut* peers = nullptr);

namespace {

using gemm::BK;
using gemm::BM;
using gemm::BN;

// ---------------------------------------------------------------------------
// Tensor maps

PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// 2-D map over a row-major matrix [outer, inner] with row pitch `ld`
// elements, box {box_inner, box_outer}, zero fill out of bounds.
int make_map(CUtensorMap* map, const void* ptr, int dtype, int64_t inner, int64_t outer, int64_t ld, int box_outer,
             int box_inner = 64, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  // A host thread that has made no runtime call yet (autograd's backward
  // thread for device 0, for one) has no current context, and the driver
  // call below needs one: bind the current device's primary context.
  int dev = 0;
  cudaGetDevice(&dev);
  cudaSetDevice(dev);
  auto enc = get_encode();
  if (!enc) return set_error(GH_ECUDA, "cuTensorMapEncodeTiled unavailable");
  const int elt = elt_size(dtype);
  if ((reinterpret_cast<uintptr_t>(ptr) & 15) || ((ld * elt) & 15))
    return set_error(GH_EUNSUPPORTED, "GEMM operand needs a 16-byte aligned base and row pitch (pitch %lld elements)",
                     (long long)ld);
  CUtensorMapDataType dt = dtype == GH_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  cuuint64_t gdim[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  cuuint64_t gstride[1] = {(cuuint64_t)(ld * elt)};
  cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, dt, 2, const_cast<void*>(ptr), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(GH_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return GH_OK;
}

int num_sms_dev() {
  int dev = 0;
  cudaGetDevice(&dev);
  static int cached[64] = {0};
  if (dev < 64 && cached[dev]) return cached[dev];
  int n = 148;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev < 64) cached[dev] = n;
  return n;
}

template <typename T, int A_MN, int B_MN, int EPI, typename OutT, int PAIR, int NSUB = 1>
int launch_gemm_t(const CUtensorMap& ta, const CUtensorMap& tb, gemm::Params& p, int max_ctas, cudaStream_t st) {
  auto kern = gemm::tc_gemm_kernel<T, A_MN, B_MN, EPI, OutT, PAIR, NSUB>;
  constexpr int SMEM = gemm::Geo<PAIR, NSUB>::SMEM;
  CUtensorMap to{};
  p.bulk_out = 0;
  if constexpr (gemm::bulk_output<EPI, OutT, NSUB>()) {
    // EPI_STORE: one output without an addend, its rows 16-byte aligned
    if (EPI != gemm::EPI_STORE ||
        (p.vec_ok && p.out && p.ksplit <= 1 && !p.split_bytes && p.npeer <= 0 && !p.add_f32 && !p.add_same)) {
      const int rc = make_map(&to, p.out, gemm::AbType<OutT>::v ? GH_BF16 : GH_F16, p.N, p.M, p.ldo, 32, 32,
                              CU_TENSOR_MAP_SWIZZLE_64B);
      if (rc) return rc;
      p.bulk_out = 1;
    }
  }
  static int max_units[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64) return set_error(GH_EUNSUPPORTED, "device index >= 64");
  if (!max_units[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return set_error(GH_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    int units = num_sms_dev() / PAIR;
    if (PAIR > 1) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 0);
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(units * PAIR);
      cfg.blockDim = dim3(gemm::THREADS);
      cfg.dynamicSmemBytes = SMEM;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = PAIR;
      at[0].val.clusterDim.y = 1;
      at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess && n > 0 && n < units) units = n;
      cudaGetLastError();
    }
    max_units[dev] = units;
  }
  int units = max_units[dev];
  if (max_ctas > 0 && max_ctas / PAIR < units) units = max_ctas / PAIR > 0 ? max_ctas / PAIR : 1;
  if (p.num_tiles < units) units = p.num_tiles;
  if (units <= 0) return GH_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * PAIR);
  cfg.blockDim = dim3(gemm::THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = PAIR;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, ta, tb, to, p);
  if (e != cudaSuccess) return set_error(GH_ECUDA, "tc_gemm launch: %s", cudaGetErrorString(e));
  count_launch(1);
  return check_launch("tc_gemm");
}

// Dispatch on majorness, pairing and tile width for a fixed (T, EPI, OutT).
template <typename T, int EPI, typename OutT>
int launch_gemm_mm(const CUtensorMap& ta, const CUtensorMap& tb, int a_mn, int b_mn, int pair, int nsub,
                   gemm::Params& p, int max_ctas, cudaStream_t st) {
  if (pair == 2 && nsub == 2) {
    if constexpr (sizeof(OutT) == 2 && EPI != gemm::EPI_LCE_Q && EPI < gemm::EPI_LSM) {
      if (p.add_f32 || p.add_same) return set_error(GH_EUNSUPPORTED, "512-column GEMM tile with an addend");
      if (!a_mn && !b_mn) return launch_gemm_t<T, 0, 0, EPI, OutT, 2, 2>(ta, tb, p, max_ctas, st);
      if (!a_mn && b_mn) return launch_gemm_t<T, 0, 1, EPI, OutT, 2, 2>(ta, tb, p, max_ctas, st);
      if (a_mn && !b_mn) return launch_gemm_t<T, 1, 0, EPI, OutT, 2, 2>(ta, tb, p, max_ctas, st);
      return launch_gemm_t<T, 1, 1, EPI, OutT, 2, 2>(ta, tb, p, max_ctas, st);
    } else {
      return set_error(GH_EUNSUPPORTED, "512-column GEMM tile with an fp32 output");
    }
  }
  if (pair == 2) {
    if (!a_mn && !b_mn) return launch_gemm_t<T, 0, 0, EPI, OutT, 2>(ta, tb, p, max_ctas, st);
    if (!a_mn && b_mn) return launch_gemm_t<T, 0, 1, EPI, OutT, 2>(ta, tb, p, max_ctas, st);
    if (a_mn && !b_mn) return launch_gemm_t<T, 1, 0, EPI, OutT, 2>(ta, tb, p, max_ctas, st);
    return launch_gemm_t<T, 1, 1, EPI, OutT, 2>(ta, tb, p, max_ctas, st);
  }
  if (!a_mn && !b_mn) return launch_gemm_t<T, 0, 0, EPI, OutT, 1>(ta, tb, p, max_ctas, st);
  if (!a_mn && b_mn) return launch_gemm_t<T, 0, 1, EPI, OutT, 1>(ta, tb, p, max_ctas, st);
  if (a_mn && !b_mn) return launch_gemm_t<T, 1, 0, EPI, OutT, 1>(ta, tb, p, max_ctas, st);
  return launch_gemm_t<T, 1, 1, EPI, OutT, 1>(ta, tb, p, max_ctas, st);
}

// 2-CTA tiles (256 rows) once there are more than 128 rows.
inline int pick_pair(int64_t M) { return M > BM ? 2 : 1; }

// Tile width of a paired GEMM: 512 columns (NSUB = 2) unless the coarser
// tiles would leave a last wave much emptier than 256-column tiles do. The
// wide tile is credited with 6 % (its measured energy saving at the power
// cap). Outputs that need an fp32 epilogue (fp32 output, an addend) keep 256
// columns: only 16-bit outputs can be parked in registers to free TMEM early.
// The linear-CE epilogue (logits + statistics, ~4k cycles per 32-column chunk
// next to the MMAs) also keeps 256 columns: with 512 the tensor pipe waited
// ~18 % of each tile for it (measured), while two 256-column accumulators
// hide it completely. GREYHOUND_B200_GEMM_WIDE=0 forces 256 columns, =2
// forces 512 wherever the output allows it.
inline int wide_mode() {
  static int mode = [] {
    const char* e = getenv("GREYHOUND_B200_GEMM_WIDE");
    return e && *e ? atoi(e) : 1;
  }();
  return mode;
}
// Tiling of one GEMM: tile width (nsub) and split-K slices (ksplit).
struct Tiling {
  int nsub = 1, ksplit = 1;
};
// Split-K (2 slices, 512-column tiles; the slices write two 16-bit partials
// that a small kernel adds) when the caller provides the second output and
// the unsplit wide tiles would leave a short last wave: dH at the Llama-3-8B
// head (8192 x 4096 output) has 256 wide tiles for 74 pair units (a 46 %
// last wave) but 512 split units (6.9 full waves). Charged 1 % for the add.
inline Tiling pick_tiling(int64_t M, int64_t N, int64_t K, int pair, int units, bool fp32_epilogue,
                          bool lce_epilogue, bool split_ok = false) {
  Tiling t;
  if (pair != 2 || N <= BN || fp32_epilogue) return t;
  const int mode = wide_mode();
  if (mode != 1) {
    t.nsub = mode == 2 ? 2 : 1;
    return t;
  }
  if (lce_epilogue) return t;
  auto eff = [&](int64_t tn, int64_t ks) {
    const int64_t tiles = ((M + 2 * BM - 1) / (2 * BM)) * ((N + tn - 1) / tn) * ks;
    const int64_t waves = (tiles + units - 1) / units;
    // useful columns per computed column (a partial last tile computes zeros)
    const double fill = (double)N / (double)(((N + tn - 1) / tn) * tn);
    return (double)tiles / (double)(waves * units) * fill;
  };
  const double narrow = eff(BN, 1), wide = eff(2 * BN, 1) * 1.06;
  // each slice keeps at least 4 stage rounds of k-steps
  const bool can_split = split_ok && (K + BK - 1) / BK >= 2 * 16;
  const double wide_split = can_split ? eff(2 * BN, 2) * 1.06 * 0.99 : 0.0;
  if (wide_split > wide * 1.02 && wide_split > narrow) {
    t.nsub = 2;
    t.ksplit = 2;
  } else if (wide >= narrow) {
    t.nsub = 2;
  }
  return t;
}
inline int pick_nsub(int64_t M, int64_t N, int pair, int units, bool fp32_epilogue, bool lce_epilogue) {
  return pick_tiling(M, N, 0, pair, units, fp32_epilogue, lce_epilogue).nsub;
}

// Tensor maps of both operands for a GEMM of M x N x K with pairing `pair`.
int make_operand_maps(CUtensorMap* ta, CUtensorMap* tb, int dtype, const Operand& A, const Operand& B, int64_t M,
                      int64_t N, int64_t K, int pair) {
  int rc;
  const int64_t ka = A.wrap ? A.wrap : K;
  if (A.mn_major) rc = make_map(ta, A.ptr, dtype, M, ka, A.ld, BK);
  else rc = make_map(ta, A.ptr, dtype, ka, M, A.ld, BM);
  if (rc) return rc;
  if (B.mn_major) rc = make_map(tb, B.ptr, dtype, N, K, B.ld, BK);
  else rc = make_map(tb, B.ptr, dtype, K, N, B.ld, BN / pair);
  return rc;
}

void set_tiles(gemm::Params& p, int64_t M, int64_t N, int64_t K, int pair, int nsub = 1, int ksplit = 1) {
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  p.num_m = (int)((M + BM * pair - 1) / (BM * pair));
  p.num_n = (int)((N + BN * nsub - 1) / (BN * nsub));
  p.ksplit = ksplit;
  p.num_tiles = p.num_m * p.num_n * ksplit;
}

// Logits GEMM tile order: groups of 16 m-tiles (4096 rows, 32 MB of H at
// D = 4096) sweep all vocab tiles before the next group starts. Measured at
// the Llama-3-8B head (ncu, DRAM read per launch): m-fastest 11.5-16 GB,
// groups of 4 / 8 / 12 / 24: 28 / 19 / 8.4 / 10 GB, groups of 16: 4.0-6.9 GB
// and 7-9 % less time. The dW GEMM keeps the n-fastest order (other orders
// and groupings read more).
constexpr int kLogitsGroup = 16;
// GREYHOUND_B200_LOGITS_GROUP overrides it (tuning sweeps)
inline int logits_group() {
  const char* e = getenv("GREYHOUND_B200_LOGITS_GROUP");
  const int g = e && *e ? atoi(e) : kLogitsGroup;
  return g >= 1 ? g : kLogitsGroup;
}
// dW / logits-style GEMMs: the 2 GB dlogits (or W) stream must not evict the
// small H operand that every tile re-reads.
constexpr Hints kStreamA_KeepB{1, 2, 1};
constexpr Hints kKeepA_StreamB{2, 1, 1};

}  // namespace
}  // namespace gh
