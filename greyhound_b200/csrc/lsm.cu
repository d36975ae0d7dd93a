// Linear selective log-softmax: log-probabilities of given tokens from hidden
// states and the head's weight, and the gradients of both for any gradient of
// the log-probabilities, without the [N, V] logits.
//
//   x[r, v] = (H[r] . W[v]) / temperature       y[r] = x[r, t] - log sum_v e^x[r, v]
//   d[r, v] = g[r] / temperature * ([v = t] - e^(x[r, v] - lse[r]))
//   dH = d W        dW = d^T H
//
// The forward is one logits GEMM whose epilogue keeps (max, sum of
// exponentials) per row and 256-column tile and the target's logit, all from
// the fp32 accumulator (tc_gemm.cuh, EPI_LSM); a combine kernel merges the
// tiles, with the last logarithm and the difference in fp64, which costs
// nothing per row.
//
// Two backward forms:
//   kept       the forward's epilogue also stores q = e^x in 16 bits. In bf16, with
//              a[r] = -g[r] / temperature * e^-lse[r], d = a (q - e^lse onehot):
//              the one-hot part goes into q's target column, a into dH's epilogue
//              and into a 16-bit copy of H for dW (up to 128 rows into two, the
//              value and its rest). Three GEMMs for both passes.
//              fp16's exponent cannot hold e^x: every 128-column group of a row is
//              stored relative to its largest value, and a pass over a chunk of
//              rows turns that into d.
//   recomputed the backward repeats the logits GEMM row chunk by row chunk with an
//              epilogue that writes d (EPI_LSM_GRAD): four GEMMs, but d for one
//              chunk of rows at a time (the caller's choice) and, over several
//              chunks, 4 D V bytes for dW's fp32 sum, where the kept form holds
//              2 N V bytes from one pass to the other.
// Bound by the tensor pipe for many rows and by reading W once for few.
#include <algorithm>
#include <cfloat>
#include <initializer_list>
#include <type_traits>

#include "row_ops.cuh"
#include "tc_gemm_host.cuh"

namespace gh {
namespace {

inline size_t al256(size_t x) { return (x + 255) & ~size_t(255); }

constexpr double kLn2d = 0.6931471805599453;
constexpr double kLog2ed = 1.4426950408889634;

// ---------------------------------------------------------------------------
// Row kernels

// Clean targets: -1 for a row that is left out, -2 for an index outside
// [0, V) (flagged; its log-probability is NaN and it has no gradient). One block
// also clears the status word first; more blocks find it cleared.
template <typename I>
__global__ void __launch_bounds__(1024)
lsm_targets_kernel(const I* __restrict__ index, int64_t rows, int64_t V, int64_t ignore, int* __restrict__ tgt,
                   int* status) {
  if (gridDim.x == 1) {
    if (threadIdx.x == 0) *status = 0;
    __syncthreads();
  }
  for (int64_t r = (int64_t)blockIdx.x * 1024 + threadIdx.x; r < rows; r += (int64_t)gridDim.x * 1024) {
    const int64_t t = (int64_t)index[r];
    const bool skip = t == ignore, bad = !skip && (t < 0 || t >= V);
    if (bad) atomicOr(status, GH_DEV_BAD_LABEL);
    tgt[r] = skip ? -1 : bad ? -2 : (int)t;
  }
}

// The last kernel of a call hands its status on to the device's sticky slot.
__device__ __forceinline__ void publish(const int* status, int* slot) {
  if (slot && blockIdx.x == 0 && threadIdx.x == 0) report_bits(slot, *reinterpret_cast<const volatile int*>(status));
}

// Logits and statistics of one or two rows: reading W once is all the time, so
// no tensor core and no 256-column tiles (501 of them on 148 SMs are 3.4 waves).
// A warp takes four vocabulary rows at a time, 8 elements of each a lane and
// step, the rows of H in shared memory as fp32; products and sums are fp32.
// Each block leaves one (max, sum) pair a row of H. The whole call at 128256 x
// 4096: 162 us for one row (1.05 GB at 6.5 TB/s) and 189 for two, where the GEMM
// takes 205; at four rows shared memory and conversions made it 226. Two blocks
// an SM with four steps of loads in flight beat more blocks with fewer.
constexpr int kFewRows = 2;
constexpr int kFewThreads = 256;
constexpr int kFewSmem = 160 * 1024;

template <typename T, int NR>
__global__ void __launch_bounds__(kFewThreads, 2)
lsm_few_rows_kernel(const T* __restrict__ H, const T* __restrict__ W, const int* __restrict__ tgt, int rows, int D,
                    int64_t V, float sc2, float2* __restrict__ stats, float* __restrict__ xt) {
  extern __shared__ __align__(16) float hs[];  // [NR][D]
  __shared__ float2 part[kFewThreads / 32][NR];
  constexpr int R = 4;
  for (int i = threadIdx.x; i < NR * D; i += kFewThreads) hs[i] = i < rows * D ? Elt<T>::to_f(H[i]) : 0.f;
  int t[NR];
#pragma unroll
  for (int k = 0; k < NR; ++k) t[k] = k < rows ? tgt[k] : -1;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // an even share of consecutive rows: 36 or 37 of 128256, where taking groups of
  // four in turn gives some warps 40 and the rest nothing to do meanwhile
  const int64_t warps = (int64_t)gridDim.x * (kFewThreads / 32), me = (int64_t)blockIdx.x * (kFewThreads / 32) + warp;
  const int64_t v1 = (me + 1) * V / warps;
  MS ms[NR];
#pragma unroll
  for (int k = 0; k < NR; ++k) ms[k] = ms_empty();
  for (int64_t v0 = me * V / warps; v0 < v1; v0 += R) {
    const int nr = v1 - v0 < R ? (int)(v1 - v0) : R;
    const T* w = W + v0 * D;
    float acc[R][NR];
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int k = 0; k < NR; ++k) acc[j][k] = 0.f;
#pragma unroll 4
    for (int d = lane * 8; d < D; d += 256) {
      Vec16<T> x[R];
#pragma unroll
      for (int j = 0; j < R; ++j)  // past the last row: the first one again, not used
        x[j].raw = ld16_last(w + (int64_t)(j < nr ? j : 0) * D + d);
      float f[R][8];
#pragma unroll
      for (int j = 0; j < R; ++j) x[j].to_float(f[j]);
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        const float4 a = *reinterpret_cast<const float4*>(hs + k * D + d);
        const float4 b = *reinterpret_cast<const float4*>(hs + k * D + d + 4);
        const float h[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int j = 0; j < R; ++j) acc[j][k] = fmaf(f[j][e], h[e], acc[j][k]);
      }
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        float s = acc[j][k];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        if (j >= nr) continue;
        if (t[k] == v0 + j && lane == 0) xt[k] = s;
        // a NaN logit has to stay in the sum
        ms[k] = s == s ? ms_fold1(ms[k], s * sc2) : MS{0.f, s};
      }
    }
  }
#pragma unroll
  for (int k = 0; k < NR; ++k)
    if (lane == 0) part[warp][k] = make_float2(ms[k].m, ms[k].s);
  __syncthreads();
  if (threadIdx.x < rows) {
    MS a = ms_empty();
    for (int i = 0; i < kFewThreads / 32; ++i) a = ms_merge(a, MS{part[i][threadIdx.x].x, part[i][threadIdx.x].y});
    stats[(int64_t)blockIdx.x * rows + threadIdx.x] = make_float2(a.m, a.s);
  }
}

struct CombineOut {
  float* y;        // [rows] log-probability of the target (0: left out)
  float* lse2;     // [rows] log-sum-exp, log2 units (may be NULL)
  float* y2;       // [rows] y once more, for the backward (may be NULL)
  // kept form only (q == NULL otherwise)
  __nv_bfloat16* q;
  int64_t ldq;
  const uint8_t* qmode;
  const float* gmax;
  float* alpha0;   // [rows] factor that turns the stored row into p - onehot; 0: left out
  const int* status;
  int* slot;       // not NULL in a call's last launch
};

// Rewrite a row that q cannot represent (a group outside the exponent window,
// a log-sum-exp outside it) as p - onehot, or zero one that is left out and
// whose values are no fit operand; by a whole block, 8 columns (of one group) a
// thread and four such vectors in flight: every row of 8192 x 128256 in 1.2 ms
// (3.7 TB/s).
__device__ __forceinline__ void lsm_fix_row(const CombineOut& o, int64_t rows, int64_t row, int flag, float l2, float y,
                                            int t) {
  uint4* q = reinterpret_cast<uint4*>(o.q + row * o.ldq);
  const int vecs = (int)(o.ldq / 8);  // the pitch: columns past V are read by nobody
  const float et = expm1f(y);
  constexpr int U = 4;
  for (int i0 = threadIdx.x; i0 < vecs; i0 += U * blockDim.x) {
    Vec16<__nv_bfloat16> v[U];
    float h[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * blockDim.x;
      v[u].raw = make_uint4(0, 0, 0, 0);
      h[u] = 0.f;
      if (i < vecs && flag == 1) {
        v[u].raw = q[i];
        const int64_t grp = (int64_t)(i >> 4) * rows + row;
        // 2^(shift - lse2) in two factors: alone it may overflow where the product does not
        h[u] = fast_exp2(0.5f * ((o.qmode[grp] ? o.gmax[grp] : 0.f) - l2));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * blockDim.x;
      if (i >= vecs) break;
      float f[8];
      v[u].to_float(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = f[k] * h[u] * h[u];  // a NaN log-sum-exp: the row's gradient is NaN
      if (flag == 1 && (t >> 3) == i) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if ((t & 7) == k) f[k] = et;
      }
      v[u].from_float(f);
      q[i] = v[u].raw;
    }
  }
}

// Merge the per-tile (max, sum) pairs of TR rows per block. The partials are
// [tile][row]: TR = 8 reads 64 bytes of 32 tiles at a time; few rows take TR = 1,
// 256 tiles at a time, whose scattered reads cost less than fewer blocks.
template <int TR>
__global__ void __launch_bounds__(256)
lsm_combine_kernel(const float2* __restrict__ stats, int num_n, int64_t rows, int64_t V, float sc2,
                   const float* __restrict__ xt, const int* __restrict__ tgt, CombineOut o) {
  constexpr int SL = 256 / TR;
  __shared__ float sm[256], ss[256];
  __shared__ int sf[256];
  const int tid = threadIdx.x, slice = tid / TR;
  const int64_t r = (int64_t)blockIdx.x * TR + tid % TR;
  MS acc = ms_empty();
  int flag = 0;
  if (r < rows) {
#pragma unroll 4
    for (int j = slice; j < num_n; j += SL) {
      const float2 p = stats[(int64_t)j * rows + r];
      acc = ms_merge(acc, MS{p.x, p.y});
      if (o.q) {
        flag |= o.qmode[((int64_t)j * 2) * rows + r];
        if ((int64_t)j * BN + BN / 2 < V) flag |= o.qmode[((int64_t)j * 2 + 1) * rows + r];
      }
    }
  }
  sm[tid] = acc.m;
  ss[tid] = acc.s;
  sf[tid] = flag;
  __syncthreads();
#pragma unroll
  for (int s = SL / 2; s > 0; s >>= 1) {
    if (slice < s) {
      const MS t = ms_merge(MS{sm[tid], ss[tid]}, MS{sm[tid + s * TR], ss[tid + s * TR]});
      sm[tid] = t.m;
      ss[tid] = t.s;
      sf[tid] |= sf[tid + s * TR];
    }
    __syncthreads();
  }
  if (slice == 0 && r < rows) {
    const double lse2 = (double)sm[tid] + log2((double)ss[tid]);
    const int t = tgt[r];
    double y = t >= 0 ? kLn2d * ((double)xt[r] * (double)sc2 - lse2) : 0.0;
    if (y > 0.0) y = 0.0;  // rounding at p = 1; a NaN stays
    o.y[r] = t == -2 ? __int_as_float(0x7fc00000) : (float)y;
    if (o.lse2) o.lse2[r] = (float)lse2;
    if (o.y2) o.y2[r] = (float)y;
    if (o.q) {
      const bool odd = sf[tid] || !(lse2 >= (double)gemm::kLsmQLo && lse2 <= (double)gemm::kLsmQHi + 32.0);
      sf[tid] = !odd ? 0 : t >= 0 ? 1 : 2;
      sm[tid] = (float)lse2;
      ss[tid] = (float)y;
      if (t < 0) {
        o.alpha0[r] = 0.f;  // must not reach the gradients, not even as 0 * NaN
      } else {
        // The target's entry of p - onehot is -(1 - p_t) = expm1(y); it outweighs
        // its row. Its 16-bit rounding would reach dW on top of the one of a * H,
        // so the row factor takes it out: alpha0 * (stored target) is exact to
        // fp32, and the row's other entries, each rounded already, move by at
        // most 2^-8.
        const double tau = expm1(y) * (odd ? 1.0 : exp2(lse2));
        const __nv_bfloat16 c = __float2bfloat16_rn((float)tau);
        const double cd = (double)__bfloat162float(c);
        const double fix = cd != 0.0 ? tau / cd : 1.0;
        o.alpha0[r] = (float)((odd ? 1.0 : exp2(-lse2)) * fix);
        if (!odd) o.q[r * o.ldq + t] = c;
      }
    }
  }
  publish(o.status, o.slot);
  if (!o.q) return;
  __syncthreads();
  for (int i = 0; i < TR; ++i) {
    const int64_t row = (int64_t)blockIdx.x * TR + i;
    if (row < rows && sf[i]) lsm_fix_row(o, rows, row, sf[i], sm[i], ss[i], tgt[row]);
  }
}

// Eight elements of the dW GEMM's second operand, in 16 bits; finite ones stay
// within +-most. With lo > 0, what the rounding took off follows lo vectors
// further on.
template <typename T>
__device__ __forceinline__ void put_operand(T* hs, int64_t i, int64_t lo, const float (&f)[8], float most) {
  float c[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) c[k] = fabsf(f[k]) <= FLT_MAX ? fminf(fmaxf(f[k], -most), most) : f[k];
  Vec16<T> v;
  v.from_float(c);
  st16(reinterpret_cast<uint4*>(hs) + i, v.raw);
  if (!lo) return;
  float r[8], rest[8];
  v.to_float(r);
#pragma unroll
  for (int k = 0; k < 8; ++k) rest[k] = fabsf(r[k]) <= 3.4e38f ? f[k] - r[k] : 0.f;  // not inf - inf
  v.from_float(rest);
  st16(reinterpret_cast<uint4*>(hs) + lo + i, v.raw);
}

// Backward, kept form: a[r] = -g[r] / temperature * alpha0[r] and a * H in 16
// bits, the dW GEMM's second operand (its rounding is dW's only one before
// the output's, and pad > 0 leaves none: two parts of `pad` rows). Left-out rows
// give exact zeros, as do those up to pad.
__global__ void __launch_bounds__(256)
lsm_rows_kernel(const __nv_bfloat16* __restrict__ H, const float* __restrict__ g, const float* __restrict__ alpha0,
                float inv_t, int64_t rows, int64_t pad, int64_t D, float* __restrict__ a_out,
                __nv_bfloat16* __restrict__ hs, int* status) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *status = 0;  // for the GEMMs that follow
  const int64_t vpr = D / 8, n = (pad ? pad : rows) * vpr, lo = pad * vpr;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / vpr;
    const float a0 = r < rows ? alpha0[r] : 0.f;
    const float a = a0 == 0.f ? 0.f : -g[r] * inv_t * a0;
    if (r < rows && i - r * vpr == 0) a_out[r] = a;
    if (!hs) continue;
    float f[8] = {};
    if (a0 != 0.f) {
      Vec16<__nv_bfloat16> v;
      v.raw = ld16(reinterpret_cast<const uint4*>(H) + i);
      v.to_float(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= a;
    }
    put_operand(hs, i, lo, f, FLT_MAX);
  }
}

// Backward, fp16: d is written times 2^k so that the largest
// row factor lies in [2^13, 2^14): (onehot - p) keeps 2^-38 of the largest
// gradient instead of fp16's 2^-24. scale = {2^k, 2^-k}; non-finite gradients
// do not count.
__global__ void __launch_bounds__(1024)
lsm_gscale_kernel(const float* __restrict__ g, const int* __restrict__ tgt, int64_t rows, float inv_t, float* scale) {
  __shared__ float sm[32];
  float m = 0.f;
  for (int64_t r = threadIdx.x; r < rows; r += 1024) {
    const float v = fabsf(g[r] * inv_t);
    if (tgt[r] >= 0 && v <= 3.4e38f) m = fmaxf(m, v);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 32; ++i) m = fmaxf(m, sm[i]);
    int k = 0;
    if (m > 0.f) k = 13 - ilogbf(m);
    k = k < -120 ? -120 : k > 120 ? 120 : k;  // both powers stay normal
    scale[0] = ldexpf(1.f, k);
    scale[1] = ldexpf(1.f, -k);
  }
}

// Row factor and target value of d for all rows. As in the kept bf16 form the
// target's entry shall not lose its row a rounding: the row is scaled by
// (rounded / exact) entry, and arow, its inverse, goes into dH's epilogue and dW's
// copy of H.
template <typename T>
__global__ void __launch_bounds__(256)
lsm_factor_kernel(const float* __restrict__ g, const float* __restrict__ y, const int* __restrict__ tgt, float inv_t,
                  const float* __restrict__ scale, int64_t rows, float* __restrict__ rfac, float* __restrict__ tval,
                  float* __restrict__ arow) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= rows) return;
  const bool on = tgt[r] >= 0;
  const float f = on ? g[r] * inv_t * (scale ? scale[0] : 1.f) : 0.f;
  const float tv = on ? -f * expm1f(y[r]) : 0.f;
  const float c = Elt<T>::to_f(Elt<T>::from_f(tv));
  // neither inf nor NaN, nor below the type's normal numbers, whose rounding is no small share of them
  constexpr float least = std::is_same<T, __half>::value ? 0x1p-14f : 1e-30f;
  const bool fit = fabsf(c) >= least && fabsf(c) <= 3.4e38f;
  rfac[r] = fit ? f * (c / tv) : f;
  tval[r] = fit ? c : tv;
  arow[r] = !on ? 0.f : fit ? tv / c : 1.f;
}

// Backward, kept form in fp16: d = rfac (onehot - q 2^(shift - lse2)), 8 columns
// at a time (of one group, whose 128 columns share a shift); grid (rows, column
// chunks). Reads and writes the chunk once: 15 us for 777 x 32003, where the GEMM
// that recomputes it takes 70.
__global__ void __launch_bounds__(256)
lsm_unpack_kernel(const __half* __restrict__ q, int64_t ldq, const float* __restrict__ gmax, int64_t N,
                  const float* __restrict__ lse2, const float* __restrict__ rfac, const float* __restrict__ tval,
                  const int* __restrict__ tgt, int64_t V, __half* __restrict__ d) {
  const int64_t r = blockIdx.x;
  const int t = tgt[r];
  const float f = rfac[r], l2 = lse2[r], tv = tval[r];
  const int64_t vecs = ldq / 8;  // the pitch: columns past V hold nothing and are read by nobody
  const __half* qr = q + r * ldq;
  __half* dr = d + r * ldq;
  for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < vecs; i += (int64_t)gridDim.y * 256) {
    Vec16<__half> v;
    if (t < 0) {
      v.raw = make_uint4(0, 0, 0, 0);  // a row left out: 0 even where q is NaN
    } else {
      v.raw = ld16_last(reinterpret_cast<const uint4*>(qr) + i);
      const float w = -f * fast_exp2(gmax[(i >> 4) * N + r] - l2);
      float x[8];
      v.to_float(x);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= w;
      if (t >> 3 == (int)i) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if ((t & 7) == k) x[k] = tv;
      }
      v.from_float(x);
    }
    st16(reinterpret_cast<uint4*>(dr) + i, v.raw);
  }
}

// arow * H with left-out rows zeroed (0 * NaN must not reach dW): the dW GEMM's
// second operand where d is written out; pad as above.
template <typename T>
__global__ void __launch_bounds__(256)
lsm_clean_rows_kernel(const T* __restrict__ H, const int* __restrict__ tgt, const float* __restrict__ arow,
                      int64_t rows, int64_t pad, int64_t vpr, T* __restrict__ out) {
  // arow is within a rounding of 1: the type's largest values may leave it, and
  // inf times an entry of d that is 0 would be NaN
  constexpr float most = std::is_same<T, __half>::value ? 65504.f : 3.3895314e38f;
  const int64_t n = (pad ? pad : rows) * vpr, lo = pad * vpr;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / vpr;
    float f[8] = {};
    if (r < rows && tgt[r] >= 0) {
      Vec16<T> v;
      v.raw = ld16(reinterpret_cast<const uint4*>(H) + i);
      const float a = arow[r];
      v.to_float(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= a;
    }
    put_operand(out, i, lo, f, most);
  }
}

// out = row[r] * scale * sum_s part[s][r][c], the slices of a split-K product.
template <typename T>
__global__ void __launch_bounds__(256)
lsm_join_kernel(const float* __restrict__ part, int slices, int64_t n, int64_t D, const float* __restrict__ row,
                const float* __restrict__ scale, T* __restrict__ out, const int* status, int* slot) {
  publish(status, slot);
  const float f = scale ? *scale : 1.f;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
    float4 a = *reinterpret_cast<const float4*>(part + i);
#pragma unroll 4
    for (int s = 1; s < slices; ++s) {
      const float4 b = *reinterpret_cast<const float4*>(part + s * n + i);
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    const float g = row ? f * row[i / D] : f;
    T o[4] = {Elt<T>::from_f(a.x * g), Elt<T>::from_f(a.y * g), Elt<T>::from_f(a.z * g), Elt<T>::from_f(a.w * g)};
    *reinterpret_cast<uint2*>(out + i) = *reinterpret_cast<const uint2*>(o);
  }
}

// ---------------------------------------------------------------------------
// Host side

// Rows of each part of the dW GEMM's second operand where it is taken in two
// parts (value and rest, one after the other along K), else 0. Up to 128 rows the
// product is bound by writing dW and a K twice as long costs little: 64 x 4096 x
// 128256 705 -> 716 us a step, 128 x 1024 x 32000 91 -> 98, and dW is 1.66e-3 off
// (its own rounding) instead of 2.35e-3; 256 x 4096 x 128256 would take 946 for 810.
int64_t dw_pad(int64_t rows) { return rows <= 128 ? (rows + BK - 1) / BK * BK : 0; }
// The dW product's K and first operand for `rows` rows of q or d.
int64_t dw_k(int64_t rows) { return dw_pad(rows) ? 2 * dw_pad(rows) : rows; }
Operand dw_operand(const void* d, int64_t ldd, int64_t rows) { return Operand{d, ldd, 1, dw_pad(rows) ? rows : 0}; }

// K slices of the dH product [rows, D] over K = V. Its few output tiles leave
// most SMs idle at a few hundred rows (512 x 1024 over 32000: 8 pair tiles for 74
// pairs of SMs, 157 us), while K is long: the slices' fp32 sums are written to
// memory and joined. Modelled in us: 0.38 a k-step of a 256 x 256 pair tile
// (measured at full load), 12 k-steps a tile for its ends, the slices' traffic
// at 5 TB/s. 0: the product is taken whole. (run_gemm's own split is of no use
// here: its two partial sums are rounded to 16 bits before they are added.)
int dh_slices(int64_t rows, int64_t D, int64_t V) {
  const int pair = pick_pair(rows);
  const int64_t units = num_sms_dev() / pair;
  const int64_t tiles = (rows + BM * pair - 1) / (BM * pair) * ((D + BN - 1) / BN);
  const int64_t nkb = (V + BK - 1) / BK;
  auto waves = [&](int64_t t) { return (double)((t + units - 1) / units); };
  double best = 0.9 * waves(tiles) * ((double)nkb + 12) * 0.38;
  int slices = 0;
  for (int s = 2; s <= 64 && nkb / s >= 8; ++s) {
    const int64_t per = (nkb + s - 1) / s, n = (nkb + per - 1) / per;  // no empty slice
    if (n != s) continue;
    const double t = waves(tiles * s) * ((double)per + 12) * 0.38 + (double)s * rows * D * 8 / 5e6 + 4.0;
    if (t < best) {
      best = t;
      slices = s;
    }
  }
  return slices;
}

// Bytes of the product's scratch: the slices in fp32.
size_t dh_scratch(int64_t rows, int64_t D, int64_t V) { return (size_t)rows * D * dh_slices(rows, D, V) * 4; }

// dH[rows, D] = row[r] * scale * (A[rows, V] W[V, D]). Where slices are joined,
// the join hands the status on to `slot`.
template <typename T>
int dh_gemm(int dtype, const Operand& A, const void* W, int64_t rows, int64_t D, int64_t V, void* out,
            const float* scale, const float* row, void* scratch, int* status, int* slot, cudaStream_t st) {
  const int slices = dh_slices(rows, D, V);
  const int sms = num_sms_dev();
  const Operand B{W, D, 1};
  if (!slices)
    return run_gemm(dtype, A, B, rows, D, V, out, dtype, D, nullptr, nullptr, 0, scale, 1, sms, st, status,
                    PROF_GEMM_DH, Hints{}, nullptr, row);
  const int pair = pick_pair(rows);
  CUtensorMap ta, tb;
  int rc = make_operand_maps(&ta, &tb, dtype, A, B, rows, D, V, pair);
  if (rc) return rc;
  gemm::Params p{};
  set_tiles(p, rows, D, V, pair, 1, slices);
  p.raster = 1;
  p.group = 1;
  p.out = scratch;
  p.ldo = D;
  p.vec_ok = 1;
  p.split_bytes = (int64_t)rows * D * 4;
  p.status = status;
  {
    ProfScope prof(PROF_GEMM_DH, st);
    rc = pair == 2 ? launch_gemm_t<T, 0, 1, gemm::EPI_STORE, float, 2>(ta, tb, p, sms, st)
                   : launch_gemm_t<T, 0, 1, gemm::EPI_STORE, float, 1>(ta, tb, p, sms, st);
    if (rc) return rc;
  }
  const int64_t n = rows * D, want = (n + 1023) / 1024, cap = 8 * (int64_t)sms;
  lsm_join_kernel<T><<<(unsigned)(want < cap ? want : cap), 256, 0, st>>>(static_cast<const float*>(scratch), slices, n,
                                                                        D, row, scale, static_cast<T*>(out), status,
                                                                        slot);
  count_launch(1);
  return check_launch("lsm_join");
}

struct FwdLayout {
  size_t status = 0, tgt, xt, lse2, stats, qmode, gmax, total;
  int64_t chunk;
  int num_n;
};

// keep: one chunk of all rows (the stored q is one operand of the backward).
FwdLayout fwd_layout(int64_t N, int64_t V, int64_t chunk, bool keep) {
  FwdLayout L;
  if (keep || chunk <= 0 || chunk > N) chunk = N;
  L.chunk = chunk;
  L.num_n = (int)((V + BN - 1) / BN);
  size_t off = 256;
  L.tgt = off;     off = al256(off + sizeof(int) * N);
  L.xt = off;      off = al256(off + sizeof(float) * chunk);
  L.lse2 = off;    off = al256(off + sizeof(float) * N);
  // the kernel for few rows leaves one pair a block, at most 8 blocks an SM
  const size_t parts = N <= kFewRows && L.num_n < 8 * num_sms_dev() ? 8 * num_sms_dev() : L.num_n;
  L.stats = off;   off = al256(off + sizeof(float2) * parts * chunk);
  L.qmode = off;   off = al256(off + (keep ? (size_t)L.num_n * 2 * chunk : 0));
  L.gmax = off;    off = al256(off + (keep ? sizeof(float) * (size_t)L.num_n * 2 * chunk : 0));
  L.total = off;
  return L;
}

// What the kept form holds between the passes: q and, in bf16, the row factors;
// in fp16 the groups' shifts and the rows' log-sum-exp, log-probability, target.
struct KeptLayout {
  size_t q = 0, alpha0 = 0, gmax = 0, lse2 = 0, y = 0, tgt = 0, total;
  int64_t ldq;
};
KeptLayout kept_layout(int64_t N, int64_t V, int dtype) {
  KeptLayout L;
  L.ldq = (V + 7) / 8 * 8;  // 16-byte row pitch for TMA
  size_t off = al256((size_t)N * L.ldq * 2);
  if (dtype == GH_BF16) {
    L.alpha0 = off; off = al256(off + sizeof(float) * N);
  } else {
    L.gmax = off;   off = al256(off + sizeof(float) * N * 2 * (size_t)((V + BN - 1) / BN));
    L.lse2 = off;   off = al256(off + sizeof(float) * N);
    L.y = off;      off = al256(off + sizeof(float) * N);
    L.tgt = off;    off = al256(off + sizeof(int) * N);
  }
  L.total = off;
  return L;
}

struct BwdLayout {
  size_t status = 0, scale = 64, tgt, rfac, tval, arow, d, hs, dh2, acc, total;
  int64_t chunk, ldd;
  bool need_acc;
};
// kept: the bf16 form that needs no d.
BwdLayout bwd_layout(int64_t N, int64_t D, int64_t V, int64_t chunk, bool kept, bool fp32_accum) {
  BwdLayout L;
  if (kept || chunk <= 0 || chunk > N) chunk = N;
  L.chunk = chunk;
  L.ldd = (V + 7) / 8 * 8;
  size_t off = 256;
  L.tgt = off;  off = al256(off + (kept ? 0 : sizeof(int) * N));
  L.rfac = off; off = al256(off + sizeof(float) * N);  // kept: a
  L.tval = off; off = al256(off + (kept ? 0 : sizeof(float) * N));
  L.arow = off; off = al256(off + (kept ? 0 : sizeof(float) * N));
  L.d = off;    off = al256(off + (kept ? 0 : (size_t)chunk * L.ldd * 2));
  // the last chunk may be shorter, be taken in two parts and in more slices of fewer rows
  const int64_t rest = N > 0 ? N - (N - 1) / chunk * chunk : 0;
  L.hs = off;   off = al256(off + (size_t)std::max(dw_k(chunk), dw_k(rest)) * D * 2);
  const size_t a = dh_scratch(chunk, D, V), b = dh_scratch(rest, D, V);
  L.dh2 = off;  off = al256(off + (a > b ? a : b));
  L.need_acc = !kept && fp32_accum && N > chunk;
  L.acc = off;
  if (L.need_acc) off = al256(off + sizeof(float) * (size_t)D * V);
  L.total = off;
  return L;
}

int targets(const void* index, int index_dtype, int64_t N, int64_t V, int64_t ignore, int* tgt, int* status,
            cudaStream_t st) {
  const unsigned grid = N <= 16384 ? 1 : (unsigned)((N + 1023) / 1024);
  if (grid > 1) cudaMemsetAsync(status, 0, sizeof(int), st);
  if (index_dtype == GH_I64)
    lsm_targets_kernel<int64_t><<<grid, 1024, 0, st>>>(static_cast<const int64_t*>(index), N, V, ignore, tgt, status);
  else
    lsm_targets_kernel<int32_t><<<grid, 1024, 0, st>>>(static_cast<const int32_t*>(index), N, V, ignore, tgt, status);
  count_launch(1);
  return check_launch("lsm_targets");
}

// One logits GEMM with a log-probability epilogue over `rows` rows.
template <typename T, int EPI>
int logits_gemm(const void* H, const void* W, int64_t rows, int64_t D, int64_t V, int dtype, gemm::Params& p,
                cudaStream_t st) {
  const int pair = pick_pair(rows);
  CUtensorMap ta, tb;
  int rc = make_operand_maps(&ta, &tb, dtype, Operand{H, D, 0}, Operand{W, D, 0}, rows, V, D, pair);
  if (rc) return rc;
  set_tiles(p, rows, V, D, pair, 1);
  p.raster = 2;
  p.group = logits_group();
  p.a_hint = kKeepA_StreamB.a;
  p.b_hint = kKeepA_StreamB.b;
  p.out_evict_first = kKeepA_StreamB.out;
  ProfScope prof(PROF_GEMM_LOGITS_CE, st);
  if (pair == 2) return launch_gemm_t<T, 0, 0, EPI, T, 2>(ta, tb, p, num_sms_dev(), st);
  return launch_gemm_t<T, 0, 0, EPI, T, 1>(ta, tb, p, num_sms_dev(), st);
}

// Blocks of lsm_few_rows_kernel, or 0 where the GEMM runs.
template <typename T, int NR>
int few_rows_blocks(int64_t D, int64_t V) {
  const size_t smem = (size_t)NR * D * sizeof(float);
  if (smem > kFewSmem) return 0;
  int dev = 0;
  cudaGetDevice(&dev);
  auto kern = lsm_few_rows_kernel<T, NR>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem) != cudaSuccess) return 0;
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, kFewThreads, smem) != cudaSuccess || per_sm < 1)
    return 0;
  const int64_t most = (V + 4 * (kFewThreads / 32) - 1) / (4 * (kFewThreads / 32));
  const int64_t blocks = (int64_t)per_sm * num_sms_dev();
  return (int)(blocks < most ? blocks : most);
}

template <typename T, int NR>
int few_rows(const void* H, const void* W, const int* tgt, int64_t rows, int64_t D, int64_t V, float sc2,
             float2* stats, int* blocks, float* xt, cudaStream_t st) {
  *blocks = few_rows_blocks<T, NR>(D, V);
  if (!*blocks) return GH_OK;
  ProfScope prof(PROF_GEMM_LOGITS_CE, st);
  lsm_few_rows_kernel<T, NR><<<*blocks, kFewThreads, (size_t)NR * D * sizeof(float), st>>>(
      static_cast<const T*>(H), static_cast<const T*>(W), tgt, (int)rows, (int)D, V, sc2, stats, xt);
  count_launch(1);
  return check_launch("lsm_few_rows");
}

int check_common(int64_t N, int64_t D, int64_t V, int dtype, int index_dtype, double inv_t) {
  if (dtype != GH_BF16 && dtype != GH_F16)
    return set_error(GH_ETYPE, "expected bf16 or fp16 operands (dtype code %d)", dtype);
  if (index_dtype != GH_I32 && index_dtype != GH_I64)
    return set_error(GH_ETYPE, "expected int32 or int64 index, got dtype code %d", index_dtype);
  if (N < 0 || D <= 0 || V <= 0 || N > INT32_MAX || V > INT32_MAX || D > INT32_MAX)
    return set_error(GH_EINVAL, "bad shape N=%lld D=%lld V=%lld", (long long)N, (long long)D, (long long)V);
  if (D % 8) return set_error(GH_EINVAL, "hidden size must be a multiple of 8 (got %lld)", (long long)D);
  if (!(inv_t > 0.0) || !(inv_t < 1e30)) return set_error(GH_EINVAL, "temperature must be positive and finite");
  return GH_OK;
}

// What vector loads, bulk copies and 8-byte stores take for granted.
int check_aligned(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15)
      return set_error(GH_EINVAL, "operands, gradients and buffers need 16-byte aligned addresses");
  return GH_OK;
}

template <typename T>
int lsm_fwd_run(const void* H, const void* W, int64_t N, int64_t D, int64_t V, int dtype, float sc2,
                const FwdLayout& L, char* kept, float* y, float* state, char* ws, cudaStream_t st) {
  constexpr bool kHalf = gemm::AbType<T>::v == 0;
  int* status = reinterpret_cast<int*>(ws + L.status);
  const KeptLayout K = kept_layout(N, V, dtype);
  const bool own_state = kHalf && kept;
  const int* tgt = reinterpret_cast<const int*>(own_state ? kept + K.tgt : ws + L.tgt);
  float* lse2 = own_state ? reinterpret_cast<float*>(kept + K.lse2) : state ? state : reinterpret_cast<float*>(ws + L.lse2);
  float* y2 = own_state ? reinterpret_cast<float*>(kept + K.y) : state ? state + N : nullptr;
  float* xt = reinterpret_cast<float*>(ws + L.xt);
  float2* stats = reinterpret_cast<float2*>(ws + L.stats);
  int* slot = nullptr;
  int rc = device_error_slot(&slot);
  if (rc) return rc;
  for (int64_t s0 = 0; s0 < N; s0 += L.chunk) {
    const int64_t rows = s0 + L.chunk <= N ? L.chunk : N - s0;
    gemm::Params p{};
    p.tgt = tgt + s0;
    p.sc2 = sc2;
    p.stats = stats;
    p.xt = xt;
    p.status = status;
    CombineOut o{};
    o.y = y + s0;
    o.lse2 = lse2 + s0;
    o.y2 = y2 ? y2 + s0 : nullptr;
    o.status = status;
    o.slot = s0 + rows >= N ? slot : nullptr;
    const void* Hc = static_cast<const T*>(H) + s0 * D;
    if (kept) {
      p.out = kept + K.q;
      p.ldo = K.ldq;
      p.vec_ok = 1;
      p.gmax = reinterpret_cast<float*>(kHalf ? kept + K.gmax : ws + L.gmax);
      if (!kHalf) {
        p.qmode = reinterpret_cast<uint8_t*>(ws + L.qmode);
        o.q = reinterpret_cast<__nv_bfloat16*>(kept + K.q);
        o.ldq = K.ldq;
        o.qmode = p.qmode;
        o.gmax = p.gmax;
        o.alpha0 = reinterpret_cast<float*>(kept + K.alpha0);
      }
      if ((rc = logits_gemm<T, gemm::EPI_LSM_Q>(Hc, W, rows, D, V, dtype, p, st))) return rc;
    }
    int parts = L.num_n;
    if (!kept) {
      int few = 0;
      if (N <= kFewRows) {
        if (N == 1) rc = few_rows<T, 1>(Hc, W, tgt + s0, rows, D, V, sc2, stats, &few, xt, st);
        else rc = few_rows<T, kFewRows>(Hc, W, tgt + s0, rows, D, V, sc2, stats, &few, xt, st);
        if (rc) return rc;
      }
      if (few) parts = few;
      else if ((rc = logits_gemm<T, gemm::EPI_LSM>(Hc, W, rows, D, V, dtype, p, st))) return rc;
    }
    // by all rows, not the chunk's: a short last chunk adds its tiles in the order
    // in which a pass that takes them all at once does
    if (N <= 4 * (int64_t)num_sms_dev())
      lsm_combine_kernel<1><<<(unsigned)rows, 256, 0, st>>>(stats, parts, rows, V, sc2, xt, tgt + s0, o);
    else
      lsm_combine_kernel<8><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(stats, parts, rows, V, sc2, xt, tgt + s0, o);
    count_launch(1);
    if ((rc = check_launch("lsm_combine"))) return rc;
  }
  if (own_state && state) {  // both were asked for: the kept buffer's copy is the caller's, too
    const cudaError_t e1 = cudaMemcpyAsync(state, lse2, sizeof(float) * N, cudaMemcpyDeviceToDevice, st);
    const cudaError_t e2 = cudaMemcpyAsync(state + N, y2, sizeof(float) * N, cudaMemcpyDeviceToDevice, st);
    if (e1 != cudaSuccess || e2 != cudaSuccess)
      return set_error(GH_ECUDA, "copy of the state: %s", cudaGetErrorString(e1 != cudaSuccess ? e1 : e2));
  }
  return GH_OK;
}

int lsm_bwd_kept_run(const void* H, const void* W, const float* grad, int64_t N, int64_t D, int64_t V, float inv_t,
                     const char* kept, void* dH, void* dW, const BwdLayout& L, char* ws, cudaStream_t st) {
  int* status = reinterpret_cast<int*>(ws + L.status);
  const KeptLayout K = kept_layout(N, V, GH_BF16);
  const int sms = num_sms_dev();
  int* slot = nullptr;
  int rc = device_error_slot(&slot);
  if (rc) return rc;
  float* a = reinterpret_cast<float*>(ws + L.rfac);
  __nv_bfloat16* hs = reinterpret_cast<__nv_bfloat16*>(ws + L.hs);
  lsm_rows_kernel<<<4 * sms, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(H), grad,
                                           reinterpret_cast<const float*>(kept + K.alpha0), inv_t, N, dw_pad(N), D, a,
                                           dW ? hs : nullptr, status);
  count_launch(1);
  if ((rc = check_launch("lsm_rows"))) return rc;
  if (dW && (rc = run_gemm(GH_BF16, dw_operand(kept + K.q, K.ldq, N), Operand{hs, D, 1}, V, D, dw_k(N), dW, GH_BF16, D,
                           nullptr, nullptr, 0, nullptr, 1, sms, st, status, PROF_GEMM_DW, kStreamA_KeepB)))
    return rc;
  if (dH && (rc = dh_gemm<__nv_bfloat16>(GH_BF16, Operand{kept + K.q, K.ldq, 0}, W, N, D, V, dH, nullptr, a,
                                         ws + L.dh2, status, slot, st)))
    return rc;
  // a joined dH has published in its last launch
  return dH && dh_slices(N, D, V) ? GH_OK : publish_status(status, st);
}

// d chunk by chunk, recomputed or (kept, fp16) from the stored q, and its products.
template <typename T>
int lsm_bwd_run(const void* H, const void* W, const int* tgt, const float* y, const float* lse2, const float* grad,
                int64_t N, int64_t D, int64_t V, int dtype, float inv_t, float sc2, const char* kept, void* dH, void* dW,
                bool fp32_accum, const BwdLayout& L, char* ws, cudaStream_t st) {
  int* status = reinterpret_cast<int*>(ws + L.status);
  const KeptLayout K = kept_layout(N, V, dtype);
  float* rfac = reinterpret_cast<float*>(ws + L.rfac);
  float* tval = reinterpret_cast<float*>(ws + L.tval);
  float* arow = reinterpret_cast<float*>(ws + L.arow);
  float* acc = reinterpret_cast<float*>(ws + L.acc);
  T* d = reinterpret_cast<T*>(ws + L.d);
  T* hs = reinterpret_cast<T*>(ws + L.hs);
  const int sms = num_sms_dev();
  const float* scale = nullptr;
  if (dtype == GH_F16) {
    float* s = reinterpret_cast<float*>(ws + L.scale);
    lsm_gscale_kernel<<<1, 1024, 0, st>>>(grad, tgt, N, inv_t, s);
    count_launch(1);
    scale = s;
  }
  lsm_factor_kernel<T><<<(unsigned)((N + 255) / 256), 256, 0, st>>>(grad, y, tgt, inv_t, scale, N, rfac, tval, arow);
  count_launch(1);
  int rc = check_launch("lsm_factor");
  if (rc) return rc;
  const float* unscale = scale ? scale + 1 : nullptr;
  for (int64_t s0 = 0; s0 < N; s0 += L.chunk) {
    const int64_t rows = s0 + L.chunk <= N ? L.chunk : N - s0;
    const bool first = s0 == 0, last = s0 + rows >= N;
    const T* Hc = static_cast<const T*>(H) + s0 * D;
    if (kept) {
      // columns shared out so that few rows fill the SMs, too
      int64_t cols = (8 * (int64_t)sms + rows - 1) / rows, most = (L.ldd / 8 + 255) / 256;
      if (cols > most) cols = most;
      if (cols > 65535) cols = 65535;
      lsm_unpack_kernel<<<dim3((unsigned)rows, (unsigned)cols), 256, 0, st>>>(
          reinterpret_cast<const __half*>(kept + K.q) + s0 * K.ldq, K.ldq,
          reinterpret_cast<const float*>(kept + K.gmax) + s0, N, lse2 + s0, rfac + s0, tval + s0, tgt + s0, V,
          reinterpret_cast<__half*>(d));
      count_launch(1);
      if ((rc = check_launch("lsm_unpack"))) return rc;
    } else {
      gemm::Params p{};
      p.tgt = tgt + s0;
      p.sc2 = sc2;
      p.lse2 = lse2 + s0;
      p.rfac = rfac + s0;
      p.tval = tval + s0;
      p.out = d;
      p.ldo = L.ldd;
      p.vec_ok = 1;
      p.status = status;
      if ((rc = logits_gemm<T, gemm::EPI_LSM_GRAD>(Hc, W, rows, D, V, dtype, p, st))) return rc;
    }
    if (dW) {
      lsm_clean_rows_kernel<T><<<4 * sms, 256, 0, st>>>(Hc, tgt + s0, arow + s0, rows, dw_pad(rows), D / 8, hs);
      count_launch(1);
      if ((rc = check_launch("lsm_clean_rows"))) return rc;
      void* out = dW;
      int out_dtype = dtype;
      const float* add_f32 = nullptr;
      const void* add_same = nullptr;
      if (L.need_acc) {
        out = last ? dW : (void*)acc;
        out_dtype = last ? dtype : GH_F32;
        add_f32 = first ? nullptr : acc;
      } else if (!fp32_accum) {
        add_same = first ? nullptr : dW;
      }
      if ((rc = run_gemm(dtype, dw_operand(d, L.ldd, rows), Operand{hs, D, 1}, V, D, dw_k(rows), out, out_dtype, D,
                         add_f32, add_same, D, unscale, 1, sms, st, status, PROF_GEMM_DW, kStreamA_KeepB)))
        return rc;
    }
    if (dH && (rc = dh_gemm<T>(dtype, Operand{d, L.ldd, 0}, W, rows, D, V, static_cast<T*>(dH) + s0 * D, unscale,
                               arow + s0, ws + L.dh2, status, nullptr, st)))
      return rc;
  }
  return publish_status(status, st);
}

}  // namespace
}  // namespace gh

using namespace gh;

extern "C" size_t gh_lsm_kept_bytes(int64_t N, int64_t V, int dtype) {
  return N < 0 || V <= 0 || elt_size(dtype) != 2 ? 0 : kept_layout(N, V, dtype).total;
}

extern "C" size_t gh_lsm_fwd_workspace_bytes(int64_t N, int64_t V, int64_t chunk_rows, int keep) {
  return N < 0 || V <= 0 ? 0 : fwd_layout(N, V, chunk_rows, keep != 0).total;
}

// A kept bf16 backward needs neither chunks nor d.
extern "C" size_t gh_lsm_bwd_workspace_bytes(int64_t N, int64_t D, int64_t V, int64_t chunk_rows, int dtype, int kept,
                                             int fp32_grad_weight_accum) {
  if (N < 0 || D <= 0 || V <= 0) return 0;
  return bwd_layout(N, D, V, chunk_rows, kept && dtype == GH_BF16, fp32_grad_weight_accum).total;
}

extern "C" int gh_lsm_fwd(const void* H, const void* W, const void* index, int index_dtype, int64_t N, int64_t D,
                          int64_t V, int dtype, int64_t ignore_index, double inv_temperature, int64_t chunk_rows,
                          float* logprobs, float* state, void* kept, size_t kept_bytes, void* workspace,
                          size_t workspace_bytes, void* stream) {
  int rc = check_common(N, D, V, dtype, index_dtype, inv_temperature);
  if (rc) return rc;
  if (N == 0) return GH_OK;
  if (!H || !W || !index || !logprobs || !workspace) return set_error(GH_EINVAL, "null pointer argument");
  if ((rc = check_aligned({H, W, kept, workspace}))) return rc;
  const KeptLayout K = kept_layout(N, V, dtype);
  if (kept && kept_bytes < K.total) return set_error(GH_EWORKSPACE, "kept buffer too small");
  const FwdLayout L = fwd_layout(N, V, chunk_rows, kept != nullptr);
  if (workspace_bytes < L.total)
    return set_error(GH_EWORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, L.total);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  char* kp = static_cast<char*>(kept);
  const float sc2 = (float)(inv_temperature * kLog2ed);
  int* status = reinterpret_cast<int*>(ws + L.status);
  int* tgt = reinterpret_cast<int*>(kp && dtype == GH_F16 ? kp + K.tgt : ws + L.tgt);
  if ((rc = targets(index, index_dtype, N, V, ignore_index, tgt, status, st))) return rc;
  if (dtype == GH_BF16) return lsm_fwd_run<__nv_bfloat16>(H, W, N, D, V, dtype, sc2, L, kp, logprobs, state, ws, st);
  return lsm_fwd_run<__half>(H, W, N, D, V, dtype, sc2, L, kp, logprobs, state, ws, st);
}

extern "C" int gh_lsm_bwd_kept(const void* H, const void* W, const float* grad, int64_t N, int64_t D, int64_t V,
                               int dtype, double inv_temperature, int64_t chunk_rows, int fp32_grad_weight_accum,
                               const void* kept, size_t kept_bytes, void* grad_input, void* grad_weight,
                               void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_common(N, D, V, dtype, GH_I64, inv_temperature);
  if (rc) return rc;
  if (N == 0) return GH_OK;
  if (!H || !W || !grad || !kept || !workspace) return set_error(GH_EINVAL, "null pointer argument");
  if ((rc = check_aligned({H, W, kept, grad_input, grad_weight, workspace}))) return rc;
  const KeptLayout K = kept_layout(N, V, dtype);
  if (kept_bytes < K.total) return set_error(GH_EWORKSPACE, "kept buffer too small");
  const BwdLayout L = bwd_layout(N, D, V, chunk_rows, dtype == GH_BF16, fp32_grad_weight_accum);
  if (workspace_bytes < L.total)
    return set_error(GH_EWORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, L.total);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const char* kp = static_cast<const char*>(kept);
  const float inv_t = (float)inv_temperature;
  if (dtype == GH_BF16)
    return lsm_bwd_kept_run(H, W, grad, N, D, V, inv_t, kp, grad_input, grad_weight, L, ws, st);
  cudaMemsetAsync(ws + L.status, 0, sizeof(int), st);
  return lsm_bwd_run<__half>(H, W, reinterpret_cast<const int*>(kp + K.tgt), reinterpret_cast<const float*>(kp + K.y),
                             reinterpret_cast<const float*>(kp + K.lse2), grad, N, D, V, dtype, inv_t, 0.f, kp,
                             grad_input, grad_weight, fp32_grad_weight_accum, L, ws, st);
}

extern "C" int gh_lsm_bwd(const void* H, const void* W, const void* index, int index_dtype, const float* state,
                          const float* grad, int64_t N, int64_t D, int64_t V, int dtype,
                          int64_t ignore_index, double inv_temperature, int64_t chunk_rows,
                          int fp32_grad_weight_accum, void* grad_input, void* grad_weight, void* workspace,
                          size_t workspace_bytes, void* stream) {
  int rc = check_common(N, D, V, dtype, index_dtype, inv_temperature);
  if (rc) return rc;
  if (N == 0) return GH_OK;
  if (!H || !W || !index || !state || !grad || !workspace)
    return set_error(GH_EINVAL, "null pointer argument");
  if ((rc = check_aligned({H, W, grad_input, grad_weight, workspace}))) return rc;
  const BwdLayout L = bwd_layout(N, D, V, chunk_rows, false, fp32_grad_weight_accum);
  if (workspace_bytes < L.total)
    return set_error(GH_EWORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, L.total);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const float inv_t = (float)inv_temperature;
  const float sc2 = (float)(inv_temperature * kLog2ed);
  const float *lse2 = state, *logprobs = state + N;
  int* status = reinterpret_cast<int*>(ws + L.status);
  int* tgt = reinterpret_cast<int*>(ws + L.tgt);
  if ((rc = targets(index, index_dtype, N, V, ignore_index, tgt, status, st))) return rc;
  if (dtype == GH_BF16)
    return lsm_bwd_run<__nv_bfloat16>(H, W, tgt, logprobs, lse2, grad, N, D, V, dtype, inv_t, sc2, nullptr, grad_input,
                                      grad_weight, fp32_grad_weight_accum, L, ws, st);
  return lsm_bwd_run<__half>(H, W, tgt, logprobs, lse2, grad, N, D, V, dtype, inv_t, sc2, nullptr, grad_input,
                             grad_weight, fp32_grad_weight_accum, L, ws, st);
}
