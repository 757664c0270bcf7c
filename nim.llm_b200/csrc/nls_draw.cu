// nls_draw.cu -- nls_draw_batch: one token per row from fp32, fp16 or bfloat16
// logits by temperature, top-k, top-p, min-p and a given uniform.
//
// The row's order is descending logits, equal ones by ascending index: token i
// has the place of comp(i) = (complement of the logit's ordered key, i), a
// 50-bit number. Every step of the definition is a prefix of that order, so
// each is the smallest comp whose running count (top-k) or running mass
// (top-p, the draw) reaches a target. No sort: the prefix is found by radix
// selection, ten bits of comp at a time, on per-bin counts or masses.
// Masses are exp((x - max) / T) in fp64, rounded to multiples of 2^-45 (at
// most 2^18 of them sum below 2^63), so sums are exact whatever their order.
#include <cmath>

#include "nls_common.cuh"
#include "nls_kernels.h"
#include "nls_types.cuh"

namespace nls {

namespace {

constexpr int kThreads = 512;
constexpr int kBinBits = 10, kBins = 1 << kBinBits;
constexpr int kIdxBits = 18;
constexpr double kUnit = 35184372088832.0;  // 2^45

struct Shared {
  unsigned long long bins[kBins];
  unsigned long long red[kThreads / 32];
  unsigned long long total;
  uint64_t lo;
  unsigned long long before;
  float fred[kThreads / 32];
  int flag;
};

template <class T>
struct Row {
  const T* x;
  int V;
  float mx;
  double inv_t;
  __device__ float val(int i) const { return to_f32(x[i]); }
  __device__ uint64_t comp(float v, int i) const { return ((uint64_t)(~fkey(v)) << kIdxBits) | (uint64_t)i; }
  // exp((x - max) / T); -inf logits have no mass
  __device__ double mass(float v) const {
    if (v == -INFINITY) return 0.0;
    return exp(((double)v - (double)mx) * inv_t);
  }
  __device__ unsigned long long units(float v) const { return __double2ull_rn(mass(v) * kUnit); }
};

__device__ unsigned long long block_sum(unsigned long long v, Shared& S) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) S.red[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long t = 0;
  for (int w = 0; w < kThreads / 32; ++w) t += S.red[w];
  return t;
}

// The smallest comp whose running count (by_count) or mass units reach
// `target` (at least one unit).
template <class T>
__device__ uint64_t find(const Row<T>& R, bool by_count, double target, Shared& S) {
  if (target < 1.0) target = 1.0;
  if (threadIdx.x == 0) {
    S.lo = 0;
    S.before = 0;
  }
  for (int shift = 50 - kBinBits; shift >= 0; shift -= kBinBits) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) S.bins[i] = 0;
    __syncthreads();
    const uint64_t lo = S.lo;
    for (int i = threadIdx.x; i < R.V; i += kThreads) {
      const float v = R.val(i);
      const uint64_t d = R.comp(v, i) - lo;
      if ((d >> (shift + kBinBits)) == 0) {
        const unsigned long long w = by_count ? 1ull : R.units(v);
        if (w) atomicAdd(&S.bins[d >> shift], w);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long c = S.before;
      int pick = -1;
      unsigned long long at = c;
      for (int b = 0; b < kBins; ++b) {
        if (S.bins[b] == 0) continue;
        pick = b;
        at = c;
        c += S.bins[b];
        if ((double)c >= target) break;
      }
      S.lo = lo + ((uint64_t)(pick < 0 ? 0 : pick) << shift);
      S.before = at;
    }
  }
  __syncthreads();
  const uint64_t r = S.lo;
  __syncthreads();
  return r;
}

template <class T>
__global__ void __launch_bounds__(kThreads) draw_kernel(const DrawArgs a) {
  __shared__ Shared S;
  const int row = blockIdx.x, tid = threadIdx.x;
  const nls_draw_params p = a.params[row];
  Row<T> R;
  R.x = static_cast<const T*>(a.logits) + (int64_t)row * a.ld;
  R.V = a.V;
  float m = -INFINITY;
  int nan = 0;
  for (int i = tid; i < a.V; i += kThreads) {
    const float v = R.val(i);
    nan |= v != v;
    m = fmaxf(m, v);
  }
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) S.fred[tid >> 5] = m;
  nan = __syncthreads_or(nan);
  for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, S.fred[w]);
  const double u = a.uniforms ? a.uniforms[row] : -1.0;
  const bool greedy = p.temperature <= 0.0;
  int err = NLS_OK;
  if (nan || isinf(m)) err = NLS_ERR_NAN_LOGITS;
  else if (!greedy && (!(p.temperature > 0.0) || !(u >= 0.0 && u < 1.0))) err = NLS_ERR_INVALID_ARG;
  if (err != NLS_OK) {
    if (tid == 0) {
      a.out_ids[row] = -1;
      if (a.out_probs) a.out_probs[row] = 0.0f;
      record_status(a.status, err);
    }
    return;
  }
  R.mx = m;
  R.inv_t = greedy ? 1.0 : fmin(1.0 / p.temperature, 1e300);
  uint64_t id;
  float prob = 1.0f;
  if (greedy || p.min_p > 1.0) {
    id = find(R, true, 1.0, S);
  } else {
    uint64_t bound = ~0ull;  // what is kept: comp <= bound
    if (p.top_k > 0 && p.top_k < a.V) bound = find(R, true, (double)p.top_k, S);
    if (p.top_p > 0.0 && p.top_p < 1.0) {
      unsigned long long t = 0;
      for (int i = tid; i < a.V; i += kThreads) {
        const float v = R.val(i);
        if (R.comp(v, i) <= bound) t += R.units(v);
      }
      const uint64_t c = find(R, false, p.top_p * (double)block_sum(t, S), S);
      if (c < bound) bound = c;
    }
    unsigned long long t = 0;
    for (int i = tid; i < a.V; i += kThreads) {
      const float v = R.val(i);
      if (R.comp(v, i) <= bound && !(p.min_p > 0.0 && R.mass(v) < p.min_p)) t += R.units(v);
    }
    const double kept = (double)block_sum(t, S);
    id = find(R, false, u * kept, S);
    prob = (float)(R.mass(R.val((int)(id & ((1u << kIdxBits) - 1)))) * kUnit / kept);
  }
  if (tid == 0) {
    a.out_ids[row] = (int64_t)(id & ((1u << kIdxBits) - 1));
    if (a.out_probs) a.out_probs[row] = prob;
  }
}

}  // namespace

cudaError_t launch_draw(const DrawArgs& a, int, cudaStream_t st) {
  with_type(a.ltype, [&](auto v) { draw_kernel<decltype(v)><<<a.rows, kThreads, 0, st>>>(a); });
  return cudaGetLastError();
}

}  // namespace nls
