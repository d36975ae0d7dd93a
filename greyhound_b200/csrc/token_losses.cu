// Losses over per-token log-probabilities: the clipped policy loss with a KL
// term, and the preference loss over pairs of sequences. Formulas with the
// kernels below.
//
// Tokens lie in sequences, either padded (T = S * L, sequence s at [s L, s L + L))
// or packed (offsets cu[0..S]); a mask may leave tokens out of both. One pass
// reads the tokens: every warp takes `span` consecutive ones and walks the
// sequences that cross them, so the work is even however the lengths are
// spread. The warp's sum over its part of sequence s goes to slot (warp + s):
// from one part to the next the warp or the sequence grows by one, so the slots
// are distinct, and at most warps + S of them exist. Sums over a sequence or
// over all then run over slots in a fixed order: no atomics, the same bits every
// time.
//
// About 20 bytes a token: HBM bound from some 10^6 tokens on, and launch
// latency below. Up to kOneBlock tokens one block does the whole forward in
// one launch.
//
// A policy term is fp32, and so is the sum of the four that a lane has at hand;
// what goes on from there is fp64 (the loss cancels: a mean of 1e-3 over a
// million terms of size 1 would keep few digits of an fp32 sum). A ratio within
// 2^-16 of a clip bound is decided in fp64. The preference sums are fp64 from the
// first difference on: they decide a whole sequence's gradient.
#include <cmath>

#include "common.cuh"

namespace gh {
namespace {

constexpr int kWarps = 8;          // warps per block, many blocks
constexpr int kOneWarps = 32;      // warps of the one block
constexpr int64_t kOneBlock = 8192;

struct Seqs {
  const void* cu;  // NULL: padded
  int cu64;
  int64_t S, L, T;
  int* slot;       // this device's error slot in pinned host memory
  int one_each;    // report sequences that do not hold exactly one token
};

__device__ __forceinline__ int64_t cu_at(const Seqs& q, int64_t s) {
  return q.cu64 ? static_cast<const int64_t*>(q.cu)[s] : (int64_t)static_cast<const int32_t*>(q.cu)[s];
}

// First token of sequence s, in [0, T] whatever the offsets hold; s in [0, S].
__device__ __forceinline__ int64_t seq_start(const Seqs& q, int64_t s) {
  if (!q.cu) return s * q.L;
  const int64_t v = cu_at(q, s);
  return v < 0 ? 0 : v > q.T ? q.T : v;
}

// The last sequence that starts at or before t; -1: t lies before them all.
__device__ __forceinline__ int64_t seq_of(const Seqs& q, int64_t t) {
  if (!q.cu) return q.L > 0 ? t / q.L : 0;
  int64_t lo = -1, hi = q.S;  // start(lo) <= t < start(hi + 1) in order
  while (lo < hi) {
    const int64_t mid = lo + (hi - lo + 1) / 2;
    if (seq_start(q, mid) <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Offsets that decrease or leave [0, T] are reported; every access stays in
// bounds all the same. Called by whole warps.
__device__ __forceinline__ void check_offsets(const Seqs& q, int64_t i, int64_t stride) {
  if (!q.cu) return;
  int bits = 0;
  for (int64_t s = i; s <= q.S; s += stride) {
    const int64_t v = cu_at(q, s), u = s > 0 ? cu_at(q, s - 1) : v;
    if (v < 0 || v > q.T || u > v) bits |= GH_DEV_BAD_SEQLENS;
    if (q.one_each && s > 0 && v != u + 1) bits |= GH_DEV_AMBIGUOUS;
  }
  bits = __reduce_or_sync(0xffffffffu, bits);  // one report a warp at most
  if ((threadIdx.x & 31) == 0) report_bits(q.slot, bits);
}

// f(s, a, b) for the parts [a, b) of [t0, t1) in token order: s in [0, S), or
// -1 for tokens that are in no sequence. Every token comes exactly once and s
// never repeats or decreases, also where the offsets are not in order. Behind a
// few empty sequences the next one that is not is searched for: a million of them
// between two tokens (offsets filled up to a fixed number) cost one warp 300 ms
// one by one. A search that offsets out of order have misled is not soon repeated.
template <typename F>
__device__ __forceinline__ void walk(const Seqs& q, int64_t t0, int64_t t1, F&& f) {
  int64_t cur = t0;
  int64_t s = cur < t1 ? seq_of(q, cur) : 0;
  int empty = 0, patience = 8;
  while (cur < t1) {
    int64_t end = s >= q.S ? t1 : seq_start(q, s + 1);
    if (end > t1) end = t1;
    if (end > cur) {
      f(s >= q.S ? (int64_t)-1 : s, cur, end);
      cur = end;
      empty = 0;
    } else if (++empty >= patience) {
      empty = 0;
      const int64_t n = seq_of(q, cur);
      if (n > s) {
        s = n;
        continue;
      }
      if (patience < 1 << 20) patience *= 2;
    }
    ++s;
  }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// Sums over a block of up to 32 warps, to every thread: K at once.
template <int K>
__device__ __forceinline__ void block_totals(double (&v)[K], double (*scratch)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = warp_sum(v[k]);
    if (lane == 0) scratch[k][warp] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(lane < warps ? scratch[k][lane] : 0.0);
}

// One sequence's (or warp's) sums.
struct Sums {
  double loss, kl;
  int64_t n;
  int clipped;  // of a warp's tokens at most
};

// ---------------------------------------------------------------------------
// Clipped policy loss
//
//   d = lp - old, r = e^d (old == NULL: r = 1)
//   pg = -min(r A, clip(r, 1 - el, 1 + eh) A)
//      = -(1 + eh) A where A > 0 and d > log(1 + eh)   (gradient 0)
//      = -(1 - el) A where A < 0 and d < log(1 - el)   (gradient 0)
//      = -r A elsewhere                                (gradient -r A)
//   u = ref - lp, kl = e^u - u - 1, dkl/dlp = -(e^u - 1)
//   l_t = pg + k kl
//   loss = sum_t l_t, or their mean over the N valid tokens, or the mean over the
//   sequences with a valid token of the mean over their valid tokens

struct Policy {
  const void *lp, *old, *ref;
  const float* adv;
  int adv_per_seq;
  const uint8_t* mask;
  double lo, hi;       // log(1 - el), log(1 + eh)
  float lo_f, hi_f;    // the same, rounded
  float at_lo, at_hi;  // 1 - el, 1 + eh
  float k;
  float* d;            // [T] gradient of l_t; NULL: not wanted
};

enum { RED_SUM = 0, RED_MEAN = 1, RED_SEQ_MEAN = 2 };

// Results of the forward. Weights of the backward: scal[0] for all tokens, or
// scal[0] / seqs[s].n.
struct PolicyOut {
  float *loss, *metrics;  // metrics: mean kl, share of clipped tokens, tokens
  float* scal;
  Sums *parts, *slots, *seqs;  // a block's (or, in the one block, a warp's) sums; (warp, sequence)'s; sequences'
};

// e^u - 1 and e^u - 1 - u. Differences of e^u would cancel at small u: the second
// comes from its Taylor series there (|u| < 1/2: the next term is below 2^-28 of
// the sum) and the first is u plus it.
__device__ __forceinline__ float kl_terms(float u, float& em1) {
  float p = 1.f / 3628800.f;
  p = fmaf(p, u, 1.f / 362880.f);
  p = fmaf(p, u, 1.f / 40320.f);
  p = fmaf(p, u, 1.f / 5040.f);
  p = fmaf(p, u, 1.f / 720.f);
  p = fmaf(p, u, 1.f / 120.f);
  p = fmaf(p, u, 1.f / 24.f);
  p = fmaf(p, u, 1.f / 6.f);
  p = fmaf(p, u, 0.5f);
  const float near = u * u * p;
  const bool small = fabsf(u) < 0.5f;
  const float far = expf(u) - 1.f;
  em1 = small ? u + near : far;
  return small ? near : far - u;
}

// The warp's tokens [t0, t1): gradients, one Sums per part (want_slots); returns
// the warp's own.
template <typename T, typename R, bool KL>
__device__ __forceinline__ Sums policy_tokens(const Seqs& q, const Policy& p, int64_t w, int64_t span, bool want_slots,
                                              const PolicyOut& o) {
  const int lane = threadIdx.x & 31;
  const T* lp = static_cast<const T*>(p.lp);
  const R* old = static_cast<const R*>(p.old);
  const R* ref = static_cast<const R*>(p.ref);
  const int64_t t0 = w * span, t1 = t0 + span < q.T ? t0 + span : q.T;
  double all_loss = 0.0, all_kl = 0.0;
  int all_clipped = 0, all_n = 0;  // of a span
  walk(q, t0, t1, [&](int64_t s, int64_t a, int64_t b) {
    if (s < 0) {
      if (p.d)
        for (int64_t t = a + lane; t < b; t += 32) p.d[t] = 0.f;
      return;
    }
    double loss = 0.0, kl = 0.0;
    int clipped = 0, valid = 0;
    // 32-bit offsets from the part's first token (a part is at most a span).
    // What is absent is read with stride 0 from an address that is there: no
    // branch stands between a lane's loads, and none of them waits for the mask.
    const int n = (int)(b - a);
    const T* lpa = lp + a;
    const R* olda = p.old ? old + a : reinterpret_cast<const R*>(p.adv);
    const R* refa = KL ? ref + a : nullptr;
    const float* adva = p.adv_per_seq ? p.adv + s : p.adv + a;
    const uint8_t* maska = p.mask ? p.mask + a : reinterpret_cast<const uint8_t*>(p.adv);
    const int olds = p.old ? 1 : 0, advs = p.adv_per_seq ? 0 : 1, masks = p.mask ? 1 : 0;
    float* da = p.d ? p.d + a : nullptr;
    constexpr int U = 4;
    for (int t = lane; t < n; t += 32 * U) {
      bool on[U];
      float x[U], y[U], z[U], av[U];
      T xr[U];
      R yr[U], zr[U];
      uint8_t mr[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = t + 32 * j < n ? t + 32 * j : t;  // past the end: the lane's first token again
        mr[j] = maska[i * masks];
        xr[j] = lpa[i];
        yr[j] = olda[i * olds];
        if (KL) zr[j] = refa[i];
        av[j] = adva[i * advs];
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        on[j] = t + 32 * j < n && (!masks || mr[j]);
        x[j] = Elt<T>::to_f(xr[j]);
        y[j] = olds ? Elt<R>::to_f(yr[j]) : x[j];
        z[j] = KL ? Elt<R>::to_f(zr[j]) : 0.f;
      }
      float l4 = 0.f, k4 = 0.f;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float g = 0.f;
        if (on[j]) {
          const float A = av[j];
          // without old the ratio is 1 even of 0 / 0; a NaN stays
          const float d = olds || x[j] != x[j] ? x[j] - y[j] : 0.f;
          bool above = d > p.hi_f, below = d < p.lo_f;
          if (fabsf(d - p.hi_f) < 0x1p-16f || fabsf(d - p.lo_f) < 0x1p-16f) {
            const double e = (double)x[j] - (double)y[j];
            above = e > p.hi;
            below = e < p.lo;
          }
          above = above && A > 0.f;
          below = below && A < 0.f;
          float l;
          if (above || below) {
            l = -A * (above ? p.at_hi : p.at_lo);
          } else {
            l = -A * expf(d);
            g = l;
          }
          if (KL) {
            float em1;
            const float k3 = kl_terms(z[j] - x[j], em1);
            if (p.k != 0.f) {  // 0 times an infinite term is no term
              g = fmaf(-p.k, em1, g);
              l = fmaf(p.k, k3, l);
            }
            k4 += k3;
          }
          l4 += l;
          clipped += above || below;
          ++valid;
        }
        if (da && t + 32 * j < n) da[t + 32 * j] = g;
      }
      loss += (double)l4;
      if (KL) kl += (double)k4;
    }
    loss = warp_sum(loss);
    if (KL) kl = warp_sum(kl);
    clipped = warp_sum(clipped);
    valid = warp_sum(valid);
    if (want_slots && lane == 0) o.slots[w + s] = Sums{loss, kl, valid, clipped};
    all_loss += loss;
    all_kl += kl;
    all_clipped += clipped;
    all_n += valid;
  });
  return Sums{all_loss, all_kl, all_n, all_clipped};
}

// Sequence s from its slots, by one warp; lane 0 writes it.
__device__ __forceinline__ void policy_sequence(const Seqs& q, int64_t s, int64_t span, const PolicyOut& o) {
  const int lane = threadIdx.x & 31;
  const int64_t a = seq_start(q, s), b = seq_start(q, s + 1);
  Sums sum{};
  double n = 0.0;
  if (b > a)
    for (int64_t w = a / span + lane; w <= (b - 1) / span; w += 32) {
      const Sums& x = o.slots[w + s];
      sum.loss += x.loss;
      n += (double)x.n;
    }
  sum.loss = warp_sum(sum.loss);
  sum.n = (int64_t)warp_sum(n);
  if (lane == 0) o.seqs[s] = sum;
}

// The last step, by one block.
__device__ __forceinline__ void policy_total(const Seqs& q, int64_t parts, int red, const PolicyOut& o) {
  __shared__ double scratch[5][32];
  double loss = 0.0, kl_sum = 0.0, clipped_sum = 0.0, n_sum = 0.0;  // counts in fp64: exact up to 2^53
  for (int64_t w = threadIdx.x; w < parts; w += blockDim.x) {
    const Sums x = o.parts[w];
    loss += x.loss;
    kl_sum += x.kl;
    clipped_sum += (double)x.clipped;
    n_sum += (double)x.n;
  }
  int filled = 0;
  if (red == RED_SEQ_MEAN) {
    loss = 0.0;
    for (int64_t s = threadIdx.x; s < q.S; s += blockDim.x) {
      const Sums x = o.seqs[s];
      if (x.n > 0) loss += x.loss / (double)x.n;
      filled += x.n > 0;
    }
  }
  double v[5] = {loss, kl_sum, clipped_sum, n_sum, (double)filled};
  block_totals(v, scratch);
  if (threadIdx.x == 0) {
    loss = v[0];
    const double kl = v[1], clipped = v[2], n = v[3];
    const double nn = n > 0 ? n : 1.0;
    double w = 1.0;
    if (red == RED_MEAN) w = 1.0 / nn;
    if (red == RED_SEQ_MEAN) w = 1.0 / (v[4] > 0 ? v[4] : 1.0);
    *o.loss = (float)(loss * w);
    o.scal[0] = (float)w;
    o.metrics[0] = (float)(kl / nn);
    o.metrics[1] = (float)(clipped / nn);
    o.metrics[2] = (float)n;
  }
}

// Four blocks an SM, so that the 32 warps an SM that cut_tokens makes run at once.
template <typename T, typename R, bool KL>
__global__ void __launch_bounds__(32 * kWarps, 4)
policy_tokens_kernel(Seqs q, Policy p, int64_t warps, int64_t span, int want_slots, PolicyOut o) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  check_offsets(q, i, (int64_t)gridDim.x * blockDim.x);
  __shared__ Sums sums[kWarps];
  Sums mine{};
  if (i / 32 < warps) mine = policy_tokens<T, R, KL>(q, p, i / 32, span, want_slots, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kWarps; ++k) {
      mine.loss += sums[k].loss;
      mine.kl += sums[k].kl;
      mine.n += sums[k].n;
      mine.clipped += sums[k].clipped;
    }
    o.parts[blockIdx.x] = mine;
  }
}
__global__ void __launch_bounds__(32 * kWarps) policy_sequences_kernel(Seqs q, int64_t span, PolicyOut o) {
  const int64_t s = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  if (s < q.S) policy_sequence(q, s, span, o);
}
__global__ void __launch_bounds__(1024) policy_total_kernel(Seqs q, int64_t parts, int red, PolicyOut o) {
  policy_total(q, parts, red, o);
}
// Everything in one block.
template <typename T, typename R, bool KL>
__global__ void __launch_bounds__(32 * kOneWarps)
policy_one_kernel(Seqs q, Policy p, int64_t warps, int64_t span, int red, PolicyOut o) {
  check_offsets(q, threadIdx.x, blockDim.x);
  const int64_t w = threadIdx.x >> 5;
  if (w < warps) {
    const Sums mine = policy_tokens<T, R, KL>(q, p, w, span, red == RED_SEQ_MEAN, o);
    if ((threadIdx.x & 31) == 0) o.parts[w] = mine;
  }
  __syncthreads();
  if (red == RED_SEQ_MEAN) {
    for (int64_t s = w; s < q.S; s += blockDim.x >> 5) policy_sequence(q, s, span, o);
    __syncthreads();
  }
  policy_total(q, warps, red, o);
}

// grad[t] = d[t] * weight * grad_output
template <typename T>
__global__ void __launch_bounds__(32 * kWarps)
policy_bwd_kernel(Seqs q, const float* __restrict__ d, const float* __restrict__ scal, const Sums* __restrict__ seqs,
                  const float* __restrict__ go, int64_t warps, int64_t span, T* __restrict__ grad) {
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  if (w >= warps) return;
  const int lane = threadIdx.x & 31;
  const float c = scal[0] * go[0];
  const int64_t t0 = w * span, t1 = t0 + span < q.T ? t0 + span : q.T;
  auto part = [&](float f, int64_t a, int64_t b) {
    const int n = (int)(b - a);
    const float* da = d + a;
    T* ga = grad + a;
    // independent loads before the first store, which may alias them for all the compiler knows
    constexpr int U = 8;
    for (int t = lane; t < n; t += 32 * U) {
      float x[U];
#pragma unroll
      for (int j = 0; j < U; ++j) x[j] = t + 32 * j < n ? da[t + 32 * j] : 0.f;
#pragma unroll
      for (int j = 0; j < U; ++j)  // a token left out stays 0 under any grad_output
        if (t + 32 * j < n) ga[t + 32 * j] = Elt<T>::from_f(x[j] == 0.f ? 0.f : x[j] * f);
    }
  };
  if (!seqs) {
    part(c, t0, t1);
    return;
  }
  walk(q, t0, t1, [&](int64_t s, int64_t a, int64_t b) {
    const int64_t n = s >= 0 ? seqs[s].n : 0;
    part(n > 0 ? c / (float)n : 0.f, a, b);
  });
}

// ---------------------------------------------------------------------------
// Preference loss
//
//   s_j = sum_t m_t (lp_t - ref_t), over n_j valid tokens; divided by n_j if
//   length-normalised. Sequences 0 .. P-1 are the chosen ones, P .. 2P-1 the
//   rejected ones, h = s_i - s_(P+i), z = beta h - margin:
//     sigmoid  (1 - e) softplus(-z) + e softplus(z)    dL/dz = e - sigmoid(-z)
//     hinge    max(0, 1 - z)                           dL/dz = -1 where z < 1
//     ipo      (h - margin - 1 / (2 beta))^2           dL/dh = 2 (h - margin - 1 / (2 beta))
//   (e: label smoothing; sigmoid'(z) terms: (1 - e)(-s(-z)) + e s(z) = e - s(-z))
//   loss = sum or mean over the pairs; dlp_t = +-(dL/dh) m_t [/ n_j] [/ P]

struct Pref {
  const void *lp, *ref;
  const uint8_t* mask;
  double beta, margin, smooth;
  int kind, normalized, mean;
};
enum { PREF_SIGMOID = 0, PREF_HINGE = 1, PREF_IPO = 2 };

struct PrefSum {
  double s;
  int64_t n;
};
struct PrefOut {
  PrefSum* slots;
  double* pair;     // [P] loss terms
  float* coef;      // [2P] gradient of a valid token
  float* rewards;   // [2P] beta s_j
  float* loss;
};

template <typename T, typename R>
__device__ __forceinline__ void pref_tokens(const Seqs& q, const Pref& p, int64_t w, int64_t span, const PrefOut& o) {
  const int lane = threadIdx.x & 31;
  const T* lp = static_cast<const T*>(p.lp);
  const R* ref = static_cast<const R*>(p.ref);
  const int64_t t0 = w * span, t1 = t0 + span < q.T ? t0 + span : q.T;
  walk(q, t0, t1, [&](int64_t s, int64_t a, int64_t b) {
    if (s < 0) return;
    double sum = 0.0;
    int n = 0;
    const int len = (int)(b - a);
    const T* lpa = lp + a;
    const R* refa = ref ? ref + a : nullptr;
    const uint8_t* maska = p.mask ? p.mask + a : nullptr;
    constexpr int U = 8;
    for (int t = lane; t < len; t += 32 * U) {
      bool on[U];
      float x[U], y[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = t + 32 * j;
        on[j] = i < len;
        x[j] = y[j] = 0.f;
        if (i < len) {  // mask or not: its load need not come first
          if (maska) on[j] = maska[i];
          x[j] = Elt<T>::to_f(lpa[i]);
          if (refa) y[j] = Elt<R>::to_f(refa[i]);
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        sum += on[j] ? (double)x[j] - (double)y[j] : 0.0;
        n += on[j];
      }
    }
    sum = warp_sum(sum);
    n = warp_sum(n);
    if (lane == 0) o.slots[w + s] = PrefSum{sum, n};
  });
}

__device__ __forceinline__ PrefSum pref_sequence(const Seqs& q, int64_t s, int64_t span, const PrefOut& o) {
  const int lane = threadIdx.x & 31;
  const int64_t a = seq_start(q, s), b = seq_start(q, s + 1);
  double sum = 0.0, n = 0.0;
  if (b > a)
    for (int64_t w = a / span + lane; w <= (b - 1) / span; w += 32) {
      const PrefSum x = o.slots[w + s];
      sum += x.s;
      n += (double)x.n;
    }
  return PrefSum{warp_sum(sum), (int64_t)warp_sum(n)};
}

__device__ __forceinline__ double softplus(double z) { return z > 0 ? z + log1p(exp(-z)) : log1p(exp(z)); }
__device__ __forceinline__ double sigmoid(double z) { return z > 0 ? 1.0 / (1.0 + exp(-z)) : exp(z) / (1.0 + exp(z)); }

// Pair i, by one warp; lane 0 writes its term.
__device__ __forceinline__ void pref_pair(const Seqs& q, const Pref& p, int64_t i, int64_t span, const PrefOut& o) {
  const int64_t P = q.S / 2;
  PrefSum c = pref_sequence(q, i, span, o), r = pref_sequence(q, P + i, span, o);
  if ((threadIdx.x & 31) != 0) return;
  const double ec = p.normalized ? 1.0 / (c.n > 0 ? (double)c.n : 1.0) : 1.0;
  const double er = p.normalized ? 1.0 / (r.n > 0 ? (double)r.n : 1.0) : 1.0;
  c.s *= ec;
  r.s *= er;
  const double h = c.s - r.s, z = p.beta * h - p.margin;
  double l, dh;
  if (p.kind == PREF_SIGMOID) {
    // a term of weight 0 may be infinite
    l = p.smooth < 1.0 ? (1.0 - p.smooth) * softplus(-z) : 0.0;
    if (p.smooth > 0.0) l += p.smooth * softplus(z);
    dh = p.beta * (p.smooth - sigmoid(-z));
  } else if (p.kind == PREF_HINGE) {
    l = z < 1.0 ? 1.0 - z : (z >= 1.0 ? 0.0 : z);  // NaN stays
    dh = z < 1.0 ? -p.beta : (z >= 1.0 ? 0.0 : z);
  } else {
    const double e = h - p.margin - 0.5 / p.beta;
    l = e * e;
    dh = 2.0 * e;
  }
  const double each = p.mean ? 1.0 / (double)P : 1.0;
  o.pair[i] = l * each;
  o.coef[i] = (float)(dh * ec * each);
  o.coef[P + i] = (float)(-dh * er * each);
  o.rewards[i] = (float)(p.beta * c.s);
  o.rewards[P + i] = (float)(p.beta * r.s);
}

__device__ __forceinline__ void pref_total(int64_t P, const PrefOut& o) {
  __shared__ double scratch[1][32];
  double l[1] = {0.0};
  for (int64_t i = threadIdx.x; i < P; i += blockDim.x) l[0] += o.pair[i];
  block_totals(l, scratch);
  if (threadIdx.x == 0) *o.loss = (float)l[0];
}

template <typename T, typename R>
__global__ void __launch_bounds__(32 * kWarps)
pref_tokens_kernel(Seqs q, Pref p, int64_t warps, int64_t span, PrefOut o) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  check_offsets(q, i, (int64_t)gridDim.x * blockDim.x);
  if (i / 32 < warps) pref_tokens<T, R>(q, p, i / 32, span, o);
}
__global__ void __launch_bounds__(32 * kWarps) pref_pairs_kernel(Seqs q, Pref p, int64_t span, PrefOut o) {
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  if (i < q.S / 2) pref_pair(q, p, i, span, o);
}
// total alone, or with the pairs in the same block
__global__ void __launch_bounds__(1024) pref_total_kernel(Seqs q, Pref p, int64_t span, int pairs_too, PrefOut o) {
  if (pairs_too) {
    for (int64_t i = threadIdx.x >> 5; i < q.S / 2; i += blockDim.x >> 5) pref_pair(q, p, i, span, o);
    __syncthreads();
  }
  pref_total(q.S / 2, o);
}
template <typename T, typename R>
__global__ void __launch_bounds__(32 * kOneWarps)
pref_one_kernel(Seqs q, Pref p, int64_t warps, int64_t span, PrefOut o) {
  check_offsets(q, threadIdx.x, blockDim.x);
  const int64_t w = threadIdx.x >> 5;
  if (w < warps) pref_tokens<T, R>(q, p, w, span, o);
  __syncthreads();
  for (int64_t i = w; i < q.S / 2; i += blockDim.x >> 5) pref_pair(q, p, i, span, o);
  __syncthreads();
  pref_total(q.S / 2, o);
}

// grad[t] = m_t coef[sequence of t] * grad_output; 0 outside the sequences.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps)
pref_bwd_kernel(Seqs q, const uint8_t* __restrict__ mask, const float* __restrict__ coef, const float* __restrict__ go,
                int64_t warps, int64_t span, T* __restrict__ grad) {
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  if (w >= warps) return;
  const int lane = threadIdx.x & 31;
  const float g = go[0];
  const int64_t t0 = w * span, t1 = t0 + span < q.T ? t0 + span : q.T;
  walk(q, t0, t1, [&](int64_t s, int64_t a, int64_t b) {
    const T v = Elt<T>::from_f(s >= 0 ? coef[s] * g : 0.f), zero = Elt<T>::from_f(0.f);
    const int n = (int)(b - a);
    T* ga = grad + a;
    const uint8_t* maska = mask ? mask + a : nullptr;
    constexpr int U = 8;
    for (int t = lane; t < n; t += 32 * U) {
      bool on[U];
#pragma unroll
      for (int j = 0; j < U; ++j) on[j] = !maska || (t + 32 * j < n && maska[t + 32 * j]);
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (t + 32 * j < n) ga[t + 32 * j] = on[j] ? v : zero;
    }
  });
}

// ---------------------------------------------------------------------------
// Host side

inline size_t al256(size_t x) { return (x + 255) & ~size_t(255); }

// How T tokens are cut: warps of `span` tokens each.
struct Cut {
  int64_t warps, span;
  bool one;
};
Cut cut_tokens(int64_t T, int64_t S, bool may_be_one) {
  Cut c;
  c.one = may_be_one && T <= kOneBlock && S <= kOneBlock;
  if (c.one) {
    c.span = (T + kOneWarps - 1) / kOneWarps;
    c.span = (c.span + 31) / 32 * 32;
  } else {
    // about 32 warps an SM; 128 tokens are one unrolled step
    c.span = (T + 148 * 32 - 1) / (148 * 32);
    c.span = (c.span + 127) / 128 * 128;
    if (c.span > 4096) c.span = 4096;
  }
  if (c.span < 32) c.span = 32;
  c.warps = (T + c.span - 1) / c.span;
  return c;
}

struct PolicyLayout {
  size_t seqs, parts, slots, total;
};
PolicyLayout policy_layout(int64_t T, int64_t S, int red) {
  const Cut c = cut_tokens(T, S, true);
  PolicyLayout L;
  size_t off = 0;
  L.seqs = off;  off = al256(off + (red == RED_SEQ_MEAN ? sizeof(Sums) * (size_t)S : 0));
  L.parts = off; off = al256(off + sizeof(Sums) * (size_t)(c.one ? kOneWarps : c.warps / kWarps + 1));
  L.slots = off; off = al256(off + (red == RED_SEQ_MEAN ? sizeof(Sums) * (size_t)(c.warps + S) : 0));
  L.total = off;
  return L;
}

struct PrefLayout {
  size_t pair, slots, total;
};
PrefLayout pref_layout(int64_t T, int64_t S) {
  const Cut c = cut_tokens(T, S, true);
  PrefLayout L;
  size_t off = 0;
  L.pair = off;  off = al256(off + sizeof(double) * (size_t)(S / 2));
  L.slots = off; off = al256(off + sizeof(PrefSum) * (size_t)(c.warps + S));
  L.total = off;
  return L;
}

inline unsigned blocks_of(int64_t warps) { return (unsigned)((warps + kWarps - 1) / kWarps); }

int make_seqs(Seqs* q, int64_t tokens, const void* cu, int cu_dtype, int64_t seqs) {
  if (tokens < 0 || seqs < 0 || tokens > ((int64_t)1 << 40) || seqs > INT32_MAX)
    return set_error(GH_EINVAL, "bad shape tokens=%lld sequences=%lld", (long long)tokens, (long long)seqs);
  if (cu && cu_dtype != GH_I32 && cu_dtype != GH_I64)
    return set_error(GH_ETYPE, "expected int32 or int64 cu_seqlens, got dtype code %d", cu_dtype);
  if (!cu && (seqs > 0 ? tokens % seqs : tokens))
    return set_error(GH_EINVAL, "%lld tokens do not divide into %lld sequences", (long long)tokens, (long long)seqs);
  q->cu = cu;
  q->cu64 = cu_dtype == GH_I64;
  q->S = seqs;
  q->L = cu || seqs == 0 ? 0 : tokens / seqs;
  q->T = tokens;
  q->slot = nullptr;
  q->one_each = 0;
  return cu ? device_error_slot(&q->slot) : GH_OK;
}

template <typename T, typename R, bool KL>
int launch_policy(const Seqs& q, const Policy& p, int red, const PolicyOut& o, cudaStream_t st) {
  const Cut c = cut_tokens(q.T, q.S, true);
  if (c.one) {
    policy_one_kernel<T, R, KL><<<1, 32 * kOneWarps, 0, st>>>(q, p, c.warps, c.span, red, o);
    count_launch(1);
    return check_launch("gh_policy_loss_fwd");
  }
  // at least one block, to check the offsets
  const unsigned grid = c.warps > 0 ? blocks_of(c.warps) : 1;
  policy_tokens_kernel<T, R, KL><<<grid, 32 * kWarps, 0, st>>>(q, p, c.warps, c.span, red == RED_SEQ_MEAN, o);
  count_launch(2);
  if (red == RED_SEQ_MEAN && q.S > 0) {
    policy_sequences_kernel<<<blocks_of(q.S), 32 * kWarps, 0, st>>>(q, c.span, o);
    count_launch(1);
  }
  policy_total_kernel<<<1, 1024, 0, st>>>(q, grid, red, o);
  return check_launch("gh_policy_loss_fwd");
}

template <typename T, typename R>
int launch_policy_kl(const Seqs& q, const Policy& p, int red, const PolicyOut& o, cudaStream_t st) {
  return p.ref ? launch_policy<T, R, true>(q, p, red, o, st) : launch_policy<T, R, false>(q, p, red, o, st);
}

template <typename T, typename R>
int launch_pref(const Seqs& q, const Pref& p, const PrefOut& o, cudaStream_t st) {
  const Cut c = cut_tokens(q.T, q.S, true);
  if (c.one) {
    pref_one_kernel<T, R><<<1, 32 * kOneWarps, 0, st>>>(q, p, c.warps, c.span, o);
    count_launch(1);
    return check_launch("gh_preference_loss_fwd");
  }
  const unsigned grid = c.warps > 0 ? blocks_of(c.warps) : 1;
  pref_tokens_kernel<T, R><<<grid, 32 * kWarps, 0, st>>>(q, p, c.warps, c.span, o);
  // few pairs: one block of 32 warps takes them and their sum (128 pairs so: 21 us,
  // against 8 in a launch of their own)
  const bool together = q.S / 2 <= 32;
  if (!together) {
    pref_pairs_kernel<<<blocks_of(q.S / 2), 32 * kWarps, 0, st>>>(q, p, c.span, o);
    count_launch(1);
  }
  pref_total_kernel<<<1, 1024, 0, st>>>(q, p, c.span, together, o);
  count_launch(2);
  return check_launch("gh_preference_loss_fwd");
}

// Dispatch on the log-probabilities' type and the other inputs' (the same, or
// fp32).
template <typename F>
int by_types(int dtype, int other, F&& f) {
  if (dtype == GH_F32 && other == GH_F32) return f(float{}, float{});
  if (dtype == GH_BF16 && other == GH_F32) return f(__nv_bfloat16{}, float{});
  if (dtype == GH_BF16 && other == GH_BF16) return f(__nv_bfloat16{}, __nv_bfloat16{});
  if (dtype == GH_F16 && other == GH_F32) return f(__half{}, float{});
  if (dtype == GH_F16 && other == GH_F16) return f(__half{}, __half{});
  return set_error(GH_ETYPE, "unsupported log-probability dtype codes %d and %d", dtype, other);
}

}  // namespace
}  // namespace gh

using namespace gh;

extern "C" size_t gh_policy_loss_workspace_bytes(int64_t tokens, int64_t seqs, int reduction) {
  return tokens < 0 || seqs < 0 ? 0 : policy_layout(tokens, seqs, reduction).total;
}

extern "C" int gh_policy_loss_fwd(const void* logprobs, int dtype, const void* old_logprobs, const void* ref_logprobs,
                                  int other_dtype, const float* advantages, int advantages_per,
                                  const uint8_t* mask, int64_t tokens, const void* cu_seqlens, int cu_dtype,
                                  int64_t seqs, double clip_low, double clip_high, double kl_multiplier, int reduction,
                                  float* loss, float* metrics, float* dlogprobs, float* scal, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  Seqs q;
  int rc = make_seqs(&q, tokens, cu_seqlens, cu_dtype, seqs);
  if (rc) return rc;
  if (reduction < RED_SUM || reduction > RED_SEQ_MEAN) return set_error(GH_EINVAL, "bad reduction %d", reduction);
  if (advantages_per < 0 || advantages_per > 2) return set_error(GH_EINVAL, "bad advantages_per %d", advantages_per);
  if (!(clip_low >= 0.0) || !(clip_high >= 0.0)) return set_error(GH_EINVAL, "clip bounds must not be negative");
  // offsets of no sequence: per-sequence advantages are empty
  if ((tokens > 0 && (!logprobs || (!advantages && seqs > 0))) || !loss || !metrics || !scal || !workspace)
    return set_error(GH_EINVAL, "null pointer argument");
  const PolicyLayout L = policy_layout(tokens, seqs, reduction);
  if (workspace_bytes < L.total)
    return set_error(GH_EWORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, L.total);
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return set_error(GH_EINVAL, "workspace must be 8-byte aligned");
  char* ws = static_cast<char*>(workspace);
  Policy p;
  p.lp = logprobs;
  p.old = old_logprobs;
  p.ref = ref_logprobs;
  p.adv = advantages;
  p.adv_per_seq = advantages_per == 1;
  q.one_each = advantages_per == 2 && cu_seqlens;
  p.mask = mask;
  p.lo = clip_low < 1.0 ? log1p(-clip_low) : -HUGE_VAL;
  p.hi = log1p(clip_high);
  p.lo_f = (float)p.lo;
  p.hi_f = (float)p.hi;
  p.at_lo = (float)(1.0 - clip_low);
  p.at_hi = (float)(1.0 + clip_high);
  p.k = (float)kl_multiplier;
  p.d = dlogprobs;
  PolicyOut o;
  o.loss = loss;
  o.metrics = metrics;
  o.scal = scal;
  o.parts = reinterpret_cast<Sums*>(ws + L.parts);
  o.slots = reinterpret_cast<Sums*>(ws + L.slots);
  o.seqs = reinterpret_cast<Sums*>(ws + L.seqs);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_types(dtype, other_dtype,
                  [&](auto t, auto r) { return launch_policy_kl<decltype(t), decltype(r)>(q, p, reduction, o, st); });
}

extern "C" int gh_policy_loss_bwd(const float* dlogprobs, const float* scal, const void* workspace,
                                  size_t workspace_bytes, const float* grad_output, int64_t tokens,
                                  const void* cu_seqlens, int cu_dtype, int64_t seqs, int reduction, void* grad,
                                  int dtype, void* stream) {
  Seqs q;
  int rc = make_seqs(&q, tokens, cu_seqlens, cu_dtype, seqs);
  if (rc) return rc;
  if (reduction < RED_SUM || reduction > RED_SEQ_MEAN) return set_error(GH_EINVAL, "bad reduction %d", reduction);
  if (tokens == 0) return GH_OK;
  if (!dlogprobs || !scal || !grad_output || !grad || !workspace) return set_error(GH_EINVAL, "null pointer argument");
  const PolicyLayout L = policy_layout(tokens, seqs, reduction);
  if (workspace_bytes < L.total) return set_error(GH_EWORKSPACE, "workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return set_error(GH_EINVAL, "workspace must be 8-byte aligned");
  const Sums* per_seq =
      reduction == RED_SEQ_MEAN ? reinterpret_cast<const Sums*>(static_cast<const char*>(workspace) + L.seqs) : nullptr;
  const Cut c = cut_tokens(tokens, seqs, false);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = by_types(dtype, GH_F32, [&](auto t, auto) {
    using T = decltype(t);
    policy_bwd_kernel<T><<<blocks_of(c.warps), 32 * kWarps, 0, st>>>(q, dlogprobs, scal, per_seq, grad_output, c.warps,
                                                                    c.span, static_cast<T*>(grad));
    count_launch(1);
    return check_launch("gh_policy_loss_bwd");
  });
  return rc;
}

extern "C" size_t gh_preference_loss_workspace_bytes(int64_t tokens, int64_t seqs) {
  return tokens < 0 || seqs < 0 ? 0 : pref_layout(tokens, seqs).total;
}

extern "C" int gh_preference_loss_fwd(const void* logprobs, int dtype, const void* ref_logprobs, int other_dtype,
                                      const uint8_t* mask, int64_t tokens, const void* cu_seqlens, int cu_dtype,
                                      int64_t seqs, double beta, double margin, double label_smoothing, int kind,
                                      int length_normalized, int mean_reduction, float* loss, float* rewards,
                                      float* coef, void* workspace, size_t workspace_bytes, void* stream) {
  Seqs q;
  int rc = make_seqs(&q, tokens, cu_seqlens, cu_dtype, seqs);
  if (rc) return rc;
  if (seqs % 2) return set_error(GH_EINVAL, "expected an even number of sequences, got %lld", (long long)seqs);
  if (kind < PREF_SIGMOID || kind > PREF_IPO) return set_error(GH_EINVAL, "bad loss kind %d", kind);
  if (!(beta > 0.0)) return set_error(GH_EINVAL, "beta must be positive");
  if ((tokens > 0 && !logprobs) || !loss || (seqs > 0 && (!rewards || !coef)) || !workspace)
    return set_error(GH_EINVAL, "null pointer argument");
  const PrefLayout L = pref_layout(tokens, seqs);
  if (workspace_bytes < L.total)
    return set_error(GH_EWORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, L.total);
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return set_error(GH_EINVAL, "workspace must be 8-byte aligned");
  char* ws = static_cast<char*>(workspace);
  Pref p;
  p.lp = logprobs;
  p.ref = ref_logprobs;
  p.mask = mask;
  p.beta = beta;
  p.margin = margin;
  p.smooth = label_smoothing;
  p.kind = kind;
  p.normalized = length_normalized;
  p.mean = mean_reduction;
  PrefOut o;
  o.slots = reinterpret_cast<PrefSum*>(ws + L.slots);
  o.pair = reinterpret_cast<double*>(ws + L.pair);
  o.coef = coef;
  o.rewards = rewards;
  o.loss = loss;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_types(dtype, other_dtype,
                  [&](auto t, auto r) { return launch_pref<decltype(t), decltype(r)>(q, p, o, st); });
}

extern "C" int gh_preference_loss_bwd(const float* coef, const float* grad_output, const uint8_t* mask, int64_t tokens,
                                      const void* cu_seqlens, int cu_dtype, int64_t seqs, void* grad, int dtype,
                                      void* stream) {
  Seqs q;
  int rc = make_seqs(&q, tokens, cu_seqlens, cu_dtype, seqs);
  if (rc) return rc;
  if (tokens == 0) return GH_OK;
  if ((seqs > 0 && !coef) || !grad_output || !grad) return set_error(GH_EINVAL, "null pointer argument");
  const Cut c = cut_tokens(tokens, seqs, false);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_types(dtype, GH_F32, [&](auto t, auto) {
    using T = decltype(t);
    pref_bwd_kernel<T><<<blocks_of(c.warps), 32 * kWarps, 0, st>>>(q, mask, coef, grad_output, c.warps, c.span,
                                                                  static_cast<T*>(grad));
    count_launch(1);
    return check_launch("gh_preference_loss_bwd");
  });
}
