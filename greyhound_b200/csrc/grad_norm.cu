// Global norm of a list of tensors, and their clipping to a largest norm.
//
//   n = sqrt(sum_i sum x^2)   or   n = max |x|      over all elements of all tensors
//   c = min(1, max_norm / (n + 1e-6));   y = c x
//
// Two launches for up to kMaxTensors tensors whatever their number and sizes:
// the list travels as a kernel argument (no copy to the device, so the calls
// can be captured), tensors are cut into chunks of kChunkBytes, and blocks
// take chunks round-robin. The first kernel leaves one partial per block; every
// block of the second sums those partials itself, in the same order, instead
// of waiting for a last block, then scales its chunks from the last one
// backwards: the end of the list is what the first pass left in L2.
//
// Bound by HBM: the norm reads every element once, at 7.2 TB/s (2.5 GB fp32 in
// 343 us); in place with c = 1 that is all (the second kernel returns), otherwise
// each is read again and written: 2.3 GB bf16, norm and scaling, in 1.06 ms,
// 6.9 GB at 6.5 TB/s.
//
// Squares are summed in fp32 over one 32-byte vector (8 or 16 terms), then in
// fp64, so a list's length costs no digits. A vector whose sum leaves
// [2^-80, 2^100] is squared again in fp64: gradients of 1e25 or 1e-25 have a
// norm, too.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "common.cuh"

namespace gh {
namespace {

constexpr int kThreads = 512;
// Four 32-byte vectors for each of a block's threads, all in flight at once
// (at two, half as much, the bf16 norm of 2.3 GB ran at 5.1 TB/s).
constexpr int64_t kChunkBytes = (int64_t)kThreads * 4 * 32;

template <int MAX>
struct List {
  const void* in[MAX];
  void* out[MAX];
  int64_t n[MAX];
  int first[MAX + 1];  // first chunk of each tensor; first[count]: their number
  uint8_t dtype[MAX];
  int count;
};
constexpr int kMaxTensors = 896;  // 32 KB of kernel arguments at most
// shorter lists cost less to hand over
constexpr int kSomeTensors = 288;
constexpr int kFewTensors = 96;
static_assert(sizeof(List<kMaxTensors>) + 128 <= 32764, "kernel arguments");

// Tensor of a chunk: the last one that starts at or before it.
template <int MAX>
__device__ __forceinline__ int tensor_of(const List<MAX>& l, int chunk) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (l.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Elements [a, b) of a tensor's chunk c. Chunks are cut where the address is a
// multiple of 32 bytes, so only a tensor's ends have scalars beside vectors.
__device__ __forceinline__ void chunk_range(const void* base, int elt, int64_t n, int64_t c, int64_t* a, int64_t* b) {
  const int64_t mis = (int64_t)(reinterpret_cast<uintptr_t>(base) & 31) / elt;
  const int64_t chunk = kChunkBytes / elt;
  int64_t s = c * chunk - mis, e = s + chunk;
  *a = s < 0 ? 0 : s;
  *b = e < n ? e : n;
}
inline int64_t chunks_of(const void* base, int elt, int64_t n) {
  const int64_t mis = (int64_t)(reinterpret_cast<uintptr_t>(base) & 31) / elt;
  return n == 0 ? 0 : ((mis + n) * elt + kChunkBytes - 1) / kChunkBytes;
}

// Accumulators: sum of squares in fp64, or the largest |x| as bits (a NaN's
// bits are above every number's, so one NaN makes the norm NaN).
struct SquareSum {
  double v = 0.0;
  template <int N>
  __device__ __forceinline__ void add(const float (&f)[N]) {
    float s = 0.f, big = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      s = fmaf(f[k], f[k], s);
      big = fmaxf(big, fabsf(f[k]));
    }
    if (s >= 0x1p-80f && s <= 0x1p100f) {
      v += (double)s;
    } else if (big > 0.f || s != s) {  // a vector of zeros adds nothing
#pragma unroll
      for (int k = 0; k < N; ++k) v += (double)f[k] * (double)f[k];
    }
  }
  __device__ __forceinline__ void add1(float f) { v += (double)f * (double)f; }
  static __device__ __forceinline__ double join(double a, double b) { return a + b; }
  __device__ __forceinline__ double value() const { return v; }
};
struct LargestAbs {
  unsigned v = 0;
  template <int N>
  __device__ __forceinline__ void add(const float (&f)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) add1(f[k]);
  }
  __device__ __forceinline__ void add1(float f) {
    const unsigned b = __float_as_uint(f) & 0x7fffffffu;
    v = b > v ? b : v;
  }
  // partials travel as the bits' value: exact in fp64, and NaN bits compare
  static __device__ __forceinline__ double join(double a, double b) { return a > b ? a : b; }
  __device__ __forceinline__ double value() const { return (double)v; }
};

template <typename A>
__device__ __forceinline__ double block_join(double v, double* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = A::join(v, __shfl_xor_sync(0xffffffffu, v, off));
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = lane < kThreads / 32 ? scratch[lane] : 0.0;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = A::join(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

template <typename T, typename A>
__device__ __forceinline__ void accumulate(const T* x, int64_t n, A& acc) {
  constexpr int PER = 32 / sizeof(T);
  constexpr int U = 4;  // 32-byte vectors in flight per thread
  const RowSplit sp = row_split(reinterpret_cast<uintptr_t>(x), n, sizeof(T), 32);
  if (threadIdx.x < sp.head) acc.add1(Elt<T>::to_f(x[threadIdx.x]));
  if (sp.tail0 + threadIdx.x < n) acc.add1(Elt<T>::to_f(x[sp.tail0 + threadIdx.x]));
  const U8* xv = reinterpret_cast<const U8*>(x + sp.head);
  int64_t i = threadIdx.x;
  for (; i + (U - 1) * kThreads < sp.nvec; i += U * kThreads) {
    Vec32<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u].raw = ld32(xv + i + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[PER];
      r[u].to_float(f);
      acc.add(f);
    }
  }
  for (; i < sp.nvec; i += kThreads) {
    Vec32<T> r;
    r.raw = ld32(xv + i);
    float f[PER];
    r.to_float(f);
    acc.add(f);
  }
}

// part[part0 + block] <- this block's share of the norm.
template <typename A, int MAX>
__global__ void __launch_bounds__(kThreads)
norm_kernel(const __grid_constant__ List<MAX> l, double* part) {
  __shared__ double scratch[kThreads / 32];
  A acc;
  for (int c = blockIdx.x; c < l.first[l.count]; c += gridDim.x) {
    const int k = tensor_of(l, c);
    const int elt = l.dtype[k] == GH_F32 ? 4 : 2;
    int64_t a, b;
    chunk_range(l.in[k], elt, l.n[k], c - l.first[k], &a, &b);
    if (l.dtype[k] == GH_F32) accumulate(static_cast<const float*>(l.in[k]) + a, b - a, acc);
    else if (l.dtype[k] == GH_BF16) accumulate(static_cast<const __nv_bfloat16*>(l.in[k]) + a, b - a, acc);
    else accumulate(static_cast<const __half*>(l.in[k]) + a, b - a, acc);
  }
  const double v = block_join<A>(acc.value(), scratch);
  if (threadIdx.x == 0) part[blockIdx.x] = v;
}

// The norm from all blocks' partials, to every thread.
template <typename A>
__device__ __forceinline__ double norm_of(const double* part, int parts, double* scratch) {
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) v = A::join(v, part[i]);
  return block_join<A>(v, scratch);
}
__device__ __forceinline__ double finish(SquareSum*, double v) { return sqrt(v); }
__device__ __forceinline__ double finish(LargestAbs*, double v) { return (double)__uint_as_float((unsigned)v); }

template <typename T>
__device__ __forceinline__ void scale_chunk(const T* x, T* y, int64_t n, float c) {
  constexpr int PER = 32 / sizeof(T);
  constexpr int U = 4;
  if ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 31) {  // no common vector boundary
    for (int64_t i = threadIdx.x; i < n; i += kThreads) y[i] = Elt<T>::from_f(Elt<T>::to_f(x[i]) * c);
    return;
  }
  const RowSplit sp = row_split(reinterpret_cast<uintptr_t>(x), n, sizeof(T), 32);
  if (threadIdx.x < sp.head) y[threadIdx.x] = Elt<T>::from_f(Elt<T>::to_f(x[threadIdx.x]) * c);
  if (sp.tail0 + threadIdx.x < n)
    y[sp.tail0 + threadIdx.x] = Elt<T>::from_f(Elt<T>::to_f(x[sp.tail0 + threadIdx.x]) * c);
  const U8* xv = reinterpret_cast<const U8*>(x + sp.head);
  U8* yv = reinterpret_cast<U8*>(y + sp.head);
  int64_t i = threadIdx.x;
  auto one = [&](Vec32<T>& r, int64_t at) {
    float f[PER];
    r.to_float(f);
#pragma unroll
    for (int k = 0; k < PER; ++k) f[k] *= c;
    r.from_float(f);
    st32_stream(yv + at, r.raw);
  };
  for (; i + (U - 1) * kThreads < sp.nvec; i += U * kThreads) {
    Vec32<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u].raw = ld32_last_rw(xv + i + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) one(r[u], i + u * kThreads);
  }
  for (; i < sp.nvec; i += kThreads) {
    Vec32<T> r;
    r.raw = ld32_last_rw(xv + i);
    one(r, i);
  }
}

// y = c x over the list; block 0 writes the norm. In place c = 1 leaves every
// element as it is; a NaN norm makes c NaN.
template <typename A, int MAX>
__global__ void __launch_bounds__(kThreads)
scale_kernel(const __grid_constant__ List<MAX> l, const double* __restrict__ part, int parts, double max_norm,
             int in_place, float* norm_out) {
  __shared__ double scratch[kThreads / 32];
  const double norm = finish((A*)nullptr, norm_of<A>(part, parts, scratch));
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) *norm_out = (float)norm;
  // no limit: nothing to scale, whatever the norm
  const double cd = max_norm == HUGE_VAL ? 1.0 : max_norm / (norm + 1e-6);
  const float c = cd >= 1.0 ? 1.f : (float)cd;
  if (in_place && c == 1.f) return;
  const int total = l.first[l.count];
  for (int j = blockIdx.x; j < total; j += gridDim.x) {
    const int ch = total - 1 - j;
    const int k = tensor_of(l, ch);
    const int elt = l.dtype[k] == GH_F32 ? 4 : 2;
    int64_t a, b;
    chunk_range(l.in[k], elt, l.n[k], ch - l.first[k], &a, &b);
    if (l.dtype[k] == GH_F32)
      scale_chunk(static_cast<const float*>(l.in[k]) + a, static_cast<float*>(l.out[k]) + a, b - a, c);
    else if (l.dtype[k] == GH_BF16)
      scale_chunk(static_cast<const __nv_bfloat16*>(l.in[k]) + a, static_cast<__nv_bfloat16*>(l.out[k]) + a, b - a, c);
    else
      scale_chunk(static_cast<const __half*>(l.in[k]) + a, static_cast<__half*>(l.out[k]) + a, b - a, c);
  }
}

// ---------------------------------------------------------------------------
// Host side

int sms() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// Tensors [*next, ...) into one list; returns the elements' chunk count or -1.
template <int MAX>
int fill(List<MAX>& l, const void* const* in, void* const* out, const int64_t* n, const int* dtype, int64_t count,
         int64_t* next) {
  l.count = 0;
  int64_t chunks = 0;
  while (*next < count && l.count < MAX) {
    const int64_t i = *next;
    const int64_t c = chunks_of(in[i], elt_size(dtype[i]), n[i]);
    if (chunks + c > INT32_MAX / 2) {
      if (l.count == 0) return -1;
      break;
    }
    ++*next;
    if (c == 0) continue;
    l.in[l.count] = in[i];
    l.out[l.count] = out ? out[i] : nullptr;
    l.n[l.count] = n[i];
    l.dtype[l.count] = (uint8_t)dtype[i];
    l.first[l.count] = (int)chunks;
    chunks += c;
    ++l.count;
  }
  l.first[l.count] = (int)chunks;
  return (int)chunks;
}

struct Call {
  const void* const* in;
  void* const* out;
  const int64_t* n;
  const int* dtype;
  int64_t count;
};

// Most blocks of one norm launch, and launches of a list.
inline int64_t norm_blocks() { return (int64_t)sms() * 4; }

template <typename A, int MAX>
int norm_lists(const Call& c, double* part, int* parts, int max_parts, cudaStream_t st) {
  int64_t next = 0;
  *parts = 0;
  while (next < c.count) {
    List<MAX> l;
    const int chunks = fill(l, c.in, nullptr, c.n, c.dtype, c.count, &next);
    if (chunks < 0) return set_error(GH_EINVAL, "a tensor has too many elements");
    if (chunks == 0) continue;
    int64_t grid = norm_blocks();
    if (grid > chunks) grid = chunks;
    if (*parts + grid > max_parts) return set_error(GH_EWORKSPACE, "workspace too small");
    norm_kernel<A, MAX><<<(unsigned)grid, kThreads, 0, st>>>(l, part + *parts);
    count_launch(1);
    *parts += (int)grid;
  }
  return check_launch("gh_global_norm");
}

template <typename A, int MAX>
int scale_lists(const Call& c, const double* part, int parts, double max_norm, int in_place, float* norm_out,
                cudaStream_t st) {
  int64_t next = 0;
  bool first = true;
  do {  // an empty list still writes its norm
    List<MAX> l;
    const int chunks = c.out ? fill(l, c.in, c.out, c.n, c.dtype, c.count, &next) : 0;
    if (!c.out) {
      l.count = 0;
      l.first[0] = 0;
      next = c.count;
    }
    if (chunks > 0 || first) {
      // twice as many blocks as the norm takes: reads and writes of 2.3 GB bf16 in
      // 0.74 ms against 0.78 (and against 0.77 with two vectors in flight, not four)
      int64_t grid = (int64_t)sms() * 8;
      if (grid > chunks) grid = chunks > 0 ? chunks : 1;
      scale_kernel<A, MAX><<<(unsigned)grid, kThreads, 0, st>>>(l, part, parts, max_norm, in_place,
                                                              first ? norm_out : nullptr);
      count_launch(1);
    }
    first = false;
  } while (next < c.count);
  return check_launch("gh_clip_by_global_norm");
}

template <typename A>
int run_call(const Call& c, double max_norm, int in_place, float* norm, double* part, int max_parts, cudaStream_t st) {
  auto both = [&](auto max) {
    constexpr int MAX = decltype(max)::value;
    int parts = 0;
    const int rc = norm_lists<A, MAX>(c, part, &parts, max_parts, st);
    return rc ? rc : scale_lists<A, MAX>(c, part, parts, max_norm, in_place, norm, st);
  };
  if (c.count <= kFewTensors) return both(std::integral_constant<int, kFewTensors>{});
  if (c.count <= kSomeTensors) return both(std::integral_constant<int, kSomeTensors>{});
  return both(std::integral_constant<int, kMaxTensors>{});
}

struct Span {
  uintptr_t a, b;
  int64_t i;
};

// Two outputs that overlap would be scaled twice or torn; an output that
// overlaps another tensor's input would change it before it is read.
int check_overlap(const Call& c) {
  std::vector<Span> o;
  o.reserve((size_t)c.count);
  for (int64_t i = 0; i < c.count; ++i)
    if (c.n[i] > 0) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(c.out[i]);
      o.push_back(Span{a, a + (uintptr_t)c.n[i] * elt_size(c.dtype[i]), i});
    }
  std::sort(o.begin(), o.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
  for (size_t k = 1; k < o.size(); ++k)
    if (o[k].a < o[k - 1].b)
      return set_error(GH_EINVAL, "tensors %lld and %lld share memory that would be scaled twice",
                       (long long)std::min(o[k].i, o[k - 1].i), (long long)std::max(o[k].i, o[k - 1].i));
  for (int64_t i = 0; i < c.count; ++i) {
    if (c.n[i] == 0 || c.in[i] == c.out[i]) continue;
    const uintptr_t a = reinterpret_cast<uintptr_t>(c.in[i]), b = a + (uintptr_t)c.n[i] * elt_size(c.dtype[i]);
    auto it = std::lower_bound(o.begin(), o.end(), b, [](const Span& x, uintptr_t v) { return x.a < v; });
    if (it != o.begin() && (it - 1)->b > a)
      return set_error(GH_EINVAL, "the output of tensor %lld overlaps the input of tensor %lld",
                       (long long)(it - 1)->i, (long long)i);
  }
  return GH_OK;
}

}  // namespace
}  // namespace gh

using namespace gh;

extern "C" size_t gh_global_norm_workspace_bytes(int64_t count) {
  if (count < 0) return 0;
  // one partial per block and launch; a launch takes kMaxTensors tensors or a
  // billion chunks
  const int64_t launches = count / kMaxTensors + 2;
  return (size_t)(launches * norm_blocks()) * sizeof(double) + 256;
}

extern "C" int gh_clip_by_global_norm(const void* const* tensors, void* const* outputs, const int64_t* numels,
                                      const int* dtypes, int64_t count, double max_norm, int inf_norm, float* norm,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  if (count < 0 || (count > 0 && (!tensors || !numels || !dtypes)) || !norm || !workspace)
    return set_error(GH_EINVAL, "null pointer argument");
  if (outputs && !(max_norm >= 0.0)) return set_error(GH_EINVAL, "max_norm must not be negative");
  int in_place = 1;
  for (int64_t i = 0; i < count; ++i) {
    if (dtypes[i] != GH_BF16 && dtypes[i] != GH_F16 && dtypes[i] != GH_F32)
      return set_error(GH_ETYPE, "unsupported dtype code %d of tensor %lld", dtypes[i], (long long)i);
    if (numels[i] < 0 || (numels[i] > 0 && (!tensors[i] || (outputs && !outputs[i]))))
      return set_error(GH_EINVAL, "bad tensor %lld", (long long)i);
    const uintptr_t at = reinterpret_cast<uintptr_t>(tensors[i]) |
                         (outputs ? reinterpret_cast<uintptr_t>(outputs[i]) : (uintptr_t)0);
    if (numels[i] > 0 && at % elt_size(dtypes[i]))
      return set_error(GH_EINVAL, "tensor %lld is not aligned to its type", (long long)i);
    if (outputs && numels[i] > 0 && outputs[i] != tensors[i]) in_place = 0;
  }
  const Call c{tensors, outputs, numels, dtypes, count};
  if (outputs) {
    try {
      const int rc = check_overlap(c);
      if (rc) return rc;
    } catch (...) {
      return set_error(GH_EINVAL, "out of host memory");
    }
  }
  if (workspace_bytes < gh_global_norm_workspace_bytes(count)) return set_error(GH_EWORKSPACE, "workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return set_error(GH_EINVAL, "workspace must be 8-byte aligned");
  double* part = static_cast<double*>(workspace);
  const int max_parts = (int)((workspace_bytes - 256) / sizeof(double));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (inf_norm) return run_call<LargestAbs>(c, max_norm, in_place, norm, part, max_parts, st);
  return run_call<SquareSum>(c, max_norm, in_place, norm, part, max_parts, st);
}
