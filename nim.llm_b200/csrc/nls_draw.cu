// nls_draw.cu -- nls_draw_batch: one token per row from fp32, fp16 or bfloat16
// logits by temperature, top-k, top-p, min-p and a given uniform.
//
// The row's order is descending logits, equal ones by ascending index: token i
// has the place of comp(i) = (complement of the logit's ordered key, i), a
// 50-bit number. Every step of the definition keeps a prefix of that order, so
// a row needs no sort: only the tokens near the borders of its prefixes do.
// Masses are exp((x - max) / T) in fp64 (a table of 64 powers of two and a
// polynomial of degree 5, after Tang, ACM TOMS 15(2), 1989; within 2^-47 of the
// value), rounded to multiples of 2^-45: at most 2^18 of them sum below 2^63,
// so their sums are exact whatever order they are added in, and a row has the
// same token whatever its batch and cluster.
//
// One thread-block cluster per row; a CTA holds its slice of the row in shared
// memory, so a logit is read from memory once. Then one of two ways:
//  * Few candidates (top-k up to 512; min-p alone): a cut that at least the
//    needed tokens reach -- for top-k a quantile of the threads' maxima, since
//    the k-th largest of some of the logits is no larger than the k-th largest
//    of all -- and the tokens above it, collected in the first CTA and sorted.
//  * Masses of the whole row (no top-k, or the candidates were too many):
//    1024 bins over the row's span of logits get their tokens' masses (and
//    counts, for top-k). The border of each prefix, and the token drawn, lie in
//    known bins; their tokens are collected and sorted.
// A bin that holds too many tokens (very many equal logits) sends the row to a
// radix selection over comp, ten bits at a time, by the first CTA alone.
// What bounds it: reading the logits for the first way; for the second the
// fp64 operations of the masses (about 13 per logit at half rate) and two
// shared-memory atomics per logit.
#include <cooperative_groups.h>

#include <cmath>

#include "nls_common.cuh"
#include "nls_kernels.h"
#include "nls_types.cuh"

namespace nls {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kBins = 1024;
constexpr int kIdxBits = 18;
constexpr int kList = 2048;           // tokens the first CTA collects and sorts
constexpr int kMine = 1024;           // tokens a CTA contributes at most
constexpr double kUnit = 35184372088832.0;  // 2^45
constexpr int kTopKMax = 512;         // top-k of the first way (16 warps x 32 maxima)
constexpr size_t kSliceBytes = 68 * 1024;  // of a CTA's slice, so that two CTAs share an SM

using u64 = unsigned long long;

// What the first CTA tells the others.
struct Command {
  int op;              // kExit, kMasses or kGather
  int r0, r1, q0, q1;  // kGather: the tokens of bins r0 .. r1 and q0 .. q1
};
constexpr int kExit = 0, kMasses = 1, kGather = 2;

struct Shared {
  u64 list[kList];
  union {
    struct {
      uint32_t lo[kBins], hi[kBins], cnt[kBins];  // this CTA's bins
    } h;
    u64 mine[kMine];                              // its tokens for the list
  };
  // of the whole row, then their running sums (first CTA)
  u64 tot[kBins];
  uint32_t tcnt[kBins];
  double pow2[64];     // 2^(j / 64)
  u64 red[kWarps];
  u64 sum[kMaxCluster], kept[kMaxCluster];  // the CTAs' masses: all, and at least min_p
  float top[kMaxCluster], low[kMaxCluster];
  int bad[kMaxCluster];
  float fred[2][kWarps];
  Command cmd;
  unsigned n_list, n_mine;
  int pick;
  u64 value;
  u64 lo;              // radix selection
  u64 before;
};

// A row's logits and settings, and the arithmetic of its masses.
struct Row {
  float mx;
  double inv_t;
  const double* pow2;
  static __device__ __forceinline__ u64 comp(float v, int i) { return ((u64)(~fkey(v)) << kIdxBits) | (u64)i; }
  static __device__ __forceinline__ float value(u64 c) { return fkey_inv(~(uint32_t)(c >> kIdxBits)); }
  // exp((v - max) / T), 0 below e^-32 (less than half a unit)
  __device__ __forceinline__ double mass(float v) const {
    const double z = __dmul_rn(__dsub_rn((double)v, (double)mx), inv_t);
    if (!(z >= -32.0)) return 0.0;  // (-inf logits too)
    const double kd = __fma_rn(z, 92.332482616893656768, 6755399441055744.0);  // z 64 / ln 2 + 1.5 2^52
    const int k = __double2loint(kd);
    const double r = __fma_rn(__dsub_rn(kd, 6755399441055744.0), -0.010830424696249145245, z);
    const double r2 = __dmul_rn(r, r);
    const double b = __fma_rn(r, 1.0 / 120.0, 1.0 / 24.0), c = __fma_rn(r, 1.0 / 6.0, 0.5);
    const double p = __fma_rn(r2, __fma_rn(r2, b, c), r);  // e^r - 1
    const double t = pow2[k & 63];
    const double s = __hiloint2double(__double2hiint(t) + ((k >> 6) << 20), __double2loint(t));
    return __fma_rn(s, p, s);
  }
  // in units of 2^-45: the low bits beside 1.5 2^7, whose last place they are
  static __device__ __forceinline__ u64 units(double m) {
    return (u64)(__double_as_longlong(__dadd_rn(m, 192.0)) - __double_as_longlong(192.0));
  }
};

__device__ u64 block_sum(u64 v, Shared& S) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) S.red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) t += S.red[w];
  return t;
}

// the running sum of v over the threads before this one
__device__ u64 block_scan(u64 v, Shared& S) {
  u64 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, o);
    if ((int)(threadIdx.x & 31) >= o) x += y;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 31) S.red[threadIdx.x >> 5] = x;
  __syncthreads();
  u64 t = x - v;
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
    if (w < (int)(threadIdx.x >> 5)) t += S.red[w];
  return t;
}

// the first bin whose running sum reaches target, or -1
template <class V>
__device__ int first_bin(const V* run, double target, Shared& S) {
  __syncthreads();
  if (threadIdx.x == 0) S.pick = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kThreads)
    if ((double)run[b] >= target && (b == 0 || (double)run[b - 1] < target)) S.pick = b;
  __syncthreads();
  return S.pick;
}

// S.list[0 .. n) ascending (n <= kList)
__device__ void sort_list(int n, Shared& S) {
  int p = 32;
  while (p < n) p <<= 1;
  for (int i = n + (int)threadIdx.x; i < p; i += kThreads) S.list[i] = ~0ull;
  __syncthreads();
  for (int size = 2; size <= p; size <<= 1) {
    for (int stride = size >> 1; stride >= 32; stride >>= 1) {
      for (int i = threadIdx.x; i < p / 2; i += kThreads) {
        const int a = ((i & ~(stride - 1)) << 1) | (i & (stride - 1)), b = a + stride;
        const u64 x = S.list[a], y = S.list[b];
        if ((x > y) == ((a & size) == 0)) {
          S.list[a] = y;
          S.list[b] = x;
        }
      }
      __syncthreads();
    }
    // strides inside 32 neighbours: one warp, in registers
    const int lane = threadIdx.x & 31;
    for (int base = 32 * (int)(threadIdx.x >> 5); base < p; base += kThreads) {
      u64 x = S.list[base + lane];
      for (int stride = min(size >> 1, 16); stride > 0; stride >>= 1) {
        const u64 y = __shfl_xor_sync(0xffffffffu, x, stride);
        const bool up = ((base + lane) & size) == 0, low = (lane & stride) == 0;
        if ((up == low) ? y < x : y > x) x = y;
      }
      S.list[base + lane] = x;
    }
    __syncthreads();
  }
}

// Radix selection over the whole row in memory: the smallest comp whose running
// count (by_count) or mass reaches target.
template <class T>
__device__ u64 select(const T* x, int V, const Row& R, bool by_count, double target, Shared& S) {
  if (target < 1.0) target = 1.0;
  if (threadIdx.x == 0) {
    S.lo = 0;
    S.before = 0;
  }
  for (int shift = 40; shift >= 0; shift -= 10) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) S.tot[i] = 0;
    __syncthreads();
    const u64 lo = S.lo, before = S.before;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float v = to_f32(x[i]);
      const u64 d = Row::comp(v, i) - lo;
      if ((d >> (shift + 10)) == 0) {
        const u64 w = by_count ? 1ull : Row::units(R.mass(v));
        if (w) atomicAdd(&S.tot[d >> shift], w);
      }
    }
    __syncthreads();
    const int b0 = 2 * threadIdx.x;
    const u64 v0 = S.tot[b0], v1 = S.tot[b0 + 1];
    const u64 e = before + block_scan(v0 + v1, S);
    __syncthreads();
    if (threadIdx.x == 0) S.pick = -1;
    __syncthreads();
    if ((double)e < target && (double)(e + v0) >= target) {
      S.pick = b0;
      S.before = e;
    } else if ((double)(e + v0) < target && (double)(e + v0 + v1) >= target) {
      S.pick = b0 + 1;
      S.before = e + v0;
    }
    __syncthreads();
    if (threadIdx.x == 0 && S.pick >= 0) S.lo = lo + ((u64)S.pick << shift);
    __syncthreads();
  }
  const u64 r = S.lo;
  __syncthreads();
  return r;
}

// The definition by radix selections, for rows that the ways above cannot take.
template <class T>
__device__ u64 draw_slowly(const T* x, int V, const Row& R, const nls_draw_params& p, double u, double* kept, Shared& S) {
  u64 bound = ~0ull;  // what is kept: comp <= bound
  if (p.top_k > 0 && p.top_k < V) bound = select(x, V, R, true, (double)p.top_k, S);
  if (p.top_p > 0.0 && p.top_p < 1.0) {
    u64 t = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float v = to_f32(x[i]);
      if (Row::comp(v, i) <= bound) t += Row::units(R.mass(v));
    }
    const u64 c = select(x, V, R, false, p.top_p * (double)block_sum(t, S), S);
    if (c < bound) bound = c;
  }
  u64 t = 0;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float v = to_f32(x[i]);
    const double m = R.mass(v);
    if (Row::comp(v, i) <= bound && !(p.min_p > 0.0 && m < p.min_p)) t += Row::units(m);
  }
  *kept = (double)block_sum(t, S);
  return select(x, V, R, false, u * *kept, S);
}

// A vector of 16 bytes as fp32.
template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  float v[N];
  __device__ __forceinline__ explicit Vec(const uint4& q) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};

template <class T>
__global__ void __launch_bounds__(kThreads) draw_kernel(const DrawArgs a, int vchunk) {
  constexpr int VN = Vec<T>::N;
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& S = *reinterpret_cast<Shared*>(smem);
  uint4* slice = reinterpret_cast<uint4*>(smem + ((sizeof(Shared) + 15) & ~size_t(15)));
  const cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)(blockIdx.x / (unsigned)C);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto remote = [&](int r) -> Shared& { return *cluster.map_shared_rank(&S, r); };

  if (tid == 0) {
    S.n_list = 0;
    S.n_mine = 0;
  }
  auto token = cluster.barrier_arrive();
  if (tid < 64) S.pow2[tid] = exp2((double)tid / 64.0);
  const nls_draw_params p = a.params[row];

  // The slice: vectors [v0, v0 + nv) of the row, counted from the 16-byte
  // boundary at or before its first logit. Vectors that reach past the row's
  // ends are read by element; what is not the row's is -inf, which is never
  // drawn and has no mass.
  const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.ld;
  const int lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int nvec = (lead + a.V + VN - 1) / VN;
  const int v0 = rank * vchunk, nv = max(0, min(vchunk, nvec - v0));
  const uint4* xv = reinterpret_cast<const uint4*>(x - lead) + v0;
  float top = -INFINITY, low = INFINITY;
  int bad = 0;
  auto take = [&](const uint4& q) {
    const Vec<T> e(q);
#pragma unroll
    for (int k = 0; k < VN; ++k) {
      bad |= e.v[k] != e.v[k];
      top = fmaxf(top, e.v[k]);
      low = fminf(low, e.v[k] == -INFINITY ? INFINITY : e.v[k]);
    }
  };
  constexpr int U = 8;  // loads in flight per thread
  for (int j = tid; j < nv; j += U * kThreads) {
    uint4 q[U];
#pragma unroll
    for (int t = 0; t < U; ++t) {
      const int i = j + t * kThreads;
      const int first = (v0 + i) * VN - lead;  // the vector's first logit
      if (i < nv && first >= 0 && first + VN <= a.V) {
        q[t] = __ldcs(xv + i);
      } else {
        union {
          T e[VN];
          uint4 v;
        } w;
#pragma unroll
        for (int k = 0; k < VN; ++k)
          w.e[k] = i < nv && first + k >= 0 && first + k < a.V ? x[first + k] : from_f32<T>(-INFINITY);
        q[t] = w.v;
      }
    }
#pragma unroll
    for (int t = 0; t < U; ++t) {
      const int i = j + t * kThreads;
      if (i < nv) slice[i] = q[t];
      take(q[t]);
    }
  }
  const float mine_top = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  if (lane == 0) {
    S.fred[0][warp] = top;
    S.fred[1][warp] = low;
  }
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    top = fmaxf(top, S.fred[0][w]);
    low = fminf(low, S.fred[1][w]);
  }
  cluster.barrier_wait(std::move(token));  // every CTA has begun
  if (tid < C) {
    Shared& D = remote(tid);
    D.top[rank] = top;
    D.low[rank] = low;
    D.bad[rank] = bad;
  }
  cluster.sync();
  for (int r = 0; r < C; ++r) {
    top = fmaxf(top, S.top[r]);
    low = fminf(low, S.low[r]);
    bad |= S.bad[r];
  }

  const double u = a.uniforms ? a.uniforms[row] : -1.0;
  const bool greedy = p.temperature <= 0.0;
  int err = NLS_OK;
  if (bad || isinf(top)) err = NLS_ERR_NAN_LOGITS;
  else if (!greedy && (!(p.temperature > 0.0) || !(u >= 0.0 && u < 1.0))) err = NLS_ERR_INVALID_ARG;
  auto finish = [&](int64_t id, float prob) {
    if (tid == 0) {
      a.out_ids[row] = id;
      if (a.out_probs) a.out_probs[row] = prob;
    }
  };
  if (err != NLS_OK) {  // (all CTAs agree; nothing remote is in flight)
    if (rank == 0) {
      finish(-1, 0.0f);
      if (tid == 0) record_status(a.status, err);
    }
    return;
  }
  Row R;
  R.mx = top;
  R.inv_t = greedy ? 1.0 : fmin(1.0 / p.temperature, 1e300);
  R.pow2 = S.pow2;
  const bool by_k = p.top_k > 0 && p.top_k < a.V, by_p = p.top_p > 0.0 && p.top_p < 1.0, by_m = p.min_p > 0.0;

  // f(logit, index) for the slice's logits above -inf
  auto each = [&](auto&& f) {
    for (int i = tid; i < nv; i += kThreads) {
      const Vec<T> e(slice[i]);
      const int first = (v0 + i) * VN - lead;
#pragma unroll
      for (int k = 0; k < VN; ++k) f(e.v[k], first + k);
    }
  };
  // The tokens that pass `want`, into the first CTA's list (its count passes
  // kList where they do not all fit). Ends with a cluster barrier.
  auto collect = [&](auto&& want) {
    __syncthreads();
    for (int i0 = 32 * warp; i0 < nv; i0 += kThreads) {
      const int i = i0 + lane;
      const uint4 none = make_uint4(0u, 0u, 0u, 0u);
      const Vec<T> e(i < nv ? slice[i] : none);
      const int first = (v0 + i) * VN - lead;
      unsigned hits = 0;
#pragma unroll
      for (int k = 0; k < VN; ++k)
        if (i < nv && e.v[k] > -INFINITY && want(e.v[k])) hits |= 1u << k;
      if (__any_sync(0xffffffffu, hits)) {
        int n = __popc(hits), at = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, at, o);
          if (lane >= o) at += y;
        }
        unsigned base = 0;
        if (lane == 31) base = atomicAdd(&S.n_mine, (unsigned)at);
        base = __shfl_sync(0xffffffffu, base, 31) + (unsigned)(at - n);
#pragma unroll
        for (int k = 0; k < VN; ++k)
          if (hits & (1u << k)) {
            if (base < kMine) S.mine[base] = Row::comp(e.v[k], first + k);
            ++base;
          }
      }
    }
    __syncthreads();
    const unsigned n = S.n_mine;
    Shared& D = remote(0);
    if (tid == 0) S.value = atomicAdd(&D.n_list, n <= kMine ? n : (unsigned)kList + 1u);
    __syncthreads();
    if (tid == 0) S.n_mine = 0;
    const unsigned at = (unsigned)S.value;
    if (n <= kMine && at + n <= kList)
      for (unsigned i = tid; i < n; i += kThreads) D.list[at + i] = S.mine[i];
    cluster.sync();
  };
  // the first CTA's next command (the others' arguments are ignored)
  auto command = [&](const Command& c) -> Command {
    if (rank == 0 && tid < C) remote(tid).cmd = c;
    cluster.sync();
    return S.cmd;
  };

  if (greedy || p.min_p > 1.0) {
    // the first of the highest logits
    unsigned best = ~0u;
    each([&](float v, int i) {
      if (v == top) best = min(best, (unsigned)i);
    });
    best = __reduce_min_sync(0xffffffffu, best);
    if (tid == 0) S.value = ~0ull;
    __syncthreads();
    if (lane == 0 && best != ~0u) atomicMin(&S.value, (u64)best);
    __syncthreads();
    if (tid == 0) remote(0).sum[rank] = S.value;
    cluster.sync();
    if (rank == 0) {
      u64 m = ~0ull;
      for (int r = 0; r < C; ++r) m = min(m, S.sum[r]);
      finish((int64_t)m, 1.0f);
    }
    return;
  }

  // ---- few candidates ---------------------------------------------------------
  if ((by_k && p.top_k <= kTopKMax) || (!by_k && !by_p && by_m)) {
    float cut;
    if (by_k) {
      // every warp's j-th largest of its threads' maxima, j = ceil(k / warps): k
      // logits of the slice reach the smallest of them (descending sort of 32;
      // the warps are those whose threads all have logits)
      const int warps = min(kWarps, nv / 32), j = warps > 0 ? ((int)p.top_k + warps - 1) / warps : 33;
      float m = mine_top;
#pragma unroll
      for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
          const float y = __shfl_xor_sync(0xffffffffu, m, stride);
          const bool down = (lane & size) == 0, lower = (lane & stride) == 0;
          m = (down == lower) ? fmaxf(m, y) : fminf(m, y);
        }
      m = __shfl_sync(0xffffffffu, m, min(j, 32) - 1);
      __syncthreads();
      if (lane == 0) S.fred[0][warp] = m;
      __syncthreads();
      cut = INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) cut = w < warps ? fminf(cut, S.fred[0][w]) : cut;
      if (j > 32) cut = -INFINITY;
    } else {
      // a little below max + T ln(min_p): the masses decide
      const double d = (double)top + p.temperature * log(p.min_p);
      const float f = (float)d;
      cut = f == f ? f - fmaxf(fabsf(f), fabsf(top)) * 0x1p-20f : -INFINITY;
    }
    collect([&](float v) { return v >= cut; });
    const unsigned n = S.n_list;
    const Command c = command(Command{n <= kList ? kExit : kMasses, 0, 0, 0, 0});
    if (c.op == kExit) {
      if (rank != 0) return;
      sort_list((int)n, S);
      int m = (int)n;  // tokens kept
      if (by_k) m = min(m, (int)p.top_k);
      // four neighbours per thread: their masses, running sums, and the steps
      u64 w[4], run[4];
      double ms[4];
      u64 t = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = 4 * tid + k;
        ms[k] = i < m ? R.mass(Row::value(S.list[i])) : 0.0;
        w[k] = Row::units(ms[k]);
        t += w[k];
        run[k] = t;
      }
      const u64 e = block_scan(t, S);
      if (tid == 0) S.value = 0;
      __syncthreads();
      if (tid == kThreads - 1) S.value = e + t;
      __syncthreads();
      const double total = (double)S.value;
      const double tp = by_p ? fmax(1.0, p.top_p * total) : 0.0;
      // kept mass: the last token with what is before it short of top-p's
      // mass, and at least min_p itself
      u64 kept = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        run[k] += e;
        const bool in = 4 * tid + k < m && (!by_p || (double)(run[k] - w[k]) < tp) && (!by_m || !(ms[k] < p.min_p));
        if (in) kept = run[k];
      }
      __syncthreads();
      if (tid == 0) S.value = 0;
      __syncthreads();
      if (kept) atomicMax(&S.value, kept);
      __syncthreads();
      const double M = (double)S.value, target = fmax(1.0, u * M);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if ((double)run[k] >= target && (double)(run[k] - w[k]) < target && 4 * tid + k < m) {
          const u64 c1 = S.list[4 * tid + k];
          a.out_ids[row] = (int64_t)(c1 & ((1u << kIdxBits) - 1));
          if (a.out_probs)
            a.out_probs[row] = (float)(exp(((double)Row::value(c1) - (double)top) * R.inv_t) * kUnit / M);
        }
      return;
    }
  }

  // ---- masses of the whole row ------------------------------------------------
  __syncthreads();
  for (int i = tid; i < kBins; i += kThreads) S.h.lo[i] = S.h.hi[i] = S.h.cnt[i] = 0;
  if (tid == 0) S.n_list = 0;
  __syncthreads();
  // logits below max - 32 T have no mass
  const float span = fminf(top - low, (float)(32.5 * p.temperature));
  const float scale = span > 0.0f ? (float)kBins / span : 0.0f;
  auto bin = [&](float v) { return min(kBins - 1, (int)((top - v) * scale)); };
  u64 all = 0, above = 0;
  each([&](float v, int) {
    const double m = R.mass(v);
    const u64 w = Row::units(m);
    all += w;
    if (by_m && !(m < p.min_p)) above += w;
    if (w) {
      const int b = bin(v);
      const uint32_t l = (uint32_t)w, was = atomicAdd(&S.h.lo[b], l);
      const uint32_t h = (uint32_t)(w >> 32) + (was + l < was ? 1u : 0u);
      if (h) atomicAdd(&S.h.hi[b], h);
      if (by_k) atomicAdd(&S.h.cnt[b], 1u);
    }
  });
  all = block_sum(all, S);
  if (by_m) above = block_sum(above, S);
  if (tid == 0) {
    Shared& D = remote(0);
    D.sum[rank] = all;
    D.kept[rank] = above;
  }
  cluster.sync();
  // each CTA adds up its share of the bins
  {
    Shared& D = remote(0);
    const int b0 = kBins * rank / C, b1 = kBins * (rank + 1) / C;
    for (int b = b0 + tid; b < b1; b += kThreads) {
      u64 t = 0;
      uint32_t n = 0;
      for (int r = 0; r < C; ++r) {
        const Shared& F = remote(r);
        t += ((u64)F.h.hi[b] << 32) + F.h.lo[b];
        if (by_k) n += F.h.cnt[b];
      }
      D.tot[b] = t;
      D.tcnt[b] = n;
    }
  }
  cluster.sync();

  if (rank != 0) {
    while (true) {
      const Command c = command(Command{});
      if (c.op == kExit) return;
      collect([&](float v) {
        const int b = bin(v);
        return ((b >= c.r0 && b <= c.r1) || (b >= c.q0 && b <= c.q1)) && Row::units(R.mass(v)) != 0;
      });
    }
  }

  // running sums of the bins (two per thread)
  {
    const u64 t0 = S.tot[2 * tid], t1 = S.tot[2 * tid + 1];
    const u64 c0 = S.tcnt[2 * tid], c1 = S.tcnt[2 * tid + 1];
    const u64 e = block_scan(t0 + t1, S);
    S.tot[2 * tid] = e + t0;
    S.tot[2 * tid + 1] = e + t0 + t1;
    if (by_k) {
      const u64 f = block_scan(c0 + c1, S);
      S.tcnt[2 * tid] = (uint32_t)(f + c0);
      S.tcnt[2 * tid + 1] = (uint32_t)(f + c0 + c1);
    }
    __syncthreads();
  }
  u64 total = 0, at_least = 0;
  for (int r = 0; r < C; ++r) {
    total += S.sum[r];
    at_least += S.kept[r];
  }
  auto before = [&](int b) -> u64 { return b > 0 ? S.tot[b - 1] : 0ull; };
  // Collects the tokens of bins r0 .. r1 and q0 .. q1 (r1 < q0, or q1 < q0 for
  // none) and sorts them; a thread's four neighbours then have their running
  // mass in the row in run[] (and themselves in S.list). False: too many.
  int n = 0;
  u64 w[4], run[4];
  auto gather = [&](int r0, int r1, int q0, int q1) -> bool {
    __syncthreads();
    if (tid == 0) S.n_list = 0;
    __syncthreads();
    (void)command(Command{kGather, r0, r1, q0, q1});
    collect([&](float v) {
      const int b = bin(v);
      return ((b >= r0 && b <= r1) || (b >= q0 && b <= q1)) && Row::units(R.mass(v)) != 0;
    });
    n = (int)S.n_list;
    if (S.n_list > kList) return false;
    sort_list(n, S);
    u64 t = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 4 * tid + k;
      w[k] = i < n ? Row::units(R.mass(Row::value(S.list[i]))) : 0;
      t += w[k];
      run[k] = t;
    }
    const u64 e = block_scan(t, S) + before(r0);
    const u64 gap = q0 <= q1 ? before(q0) - S.tot[r1] : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 4 * tid + k;
      run[k] += e;
      if (i < n && q0 <= q1 && bin(Row::value(S.list[i])) >= q0) run[k] += gap;
    }
    return true;
  };
  // the collected token whose running mass is the first to reach target: its
  // place in the list, and that mass in S.value
  auto reach = [&](double target) -> int {
    __syncthreads();
    if (tid == 0) S.pick = -1;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (4 * tid + k < n && (double)run[k] >= target && (double)(run[k] - w[k]) < target) {
        S.pick = 4 * tid + k;
        S.value = run[k];
      }
    __syncthreads();
    return S.pick;
  };

  bool ok = true;
  if (by_k) {
    const int b = first_bin(S.tcnt, (double)p.top_k, S);
    if (b >= 0) {  // (else all tokens with a mass are kept)
      ok = gather(b, b, 0, -1);
      if (ok) {
        const int i = (int)(p.top_k - 1) - (b > 0 ? (int)S.tcnt[b - 1] : 0);
        __syncthreads();
        if (i / 4 == tid) S.value = run[i & 3];
        __syncthreads();
        total = S.value;
      }
    }
  }
  u64 kept = by_m && at_least < total ? at_least : total;
  int i = -1;
  double M = (double)kept;
  if (ok && by_p) {
    const double tp = fmax(1.0, p.top_p * (double)total);
    const int b = first_bin(S.tot, tp, S);
    // the kept mass lies in bin b: so does, mostly, the drawn token's bin
    const double m0 = fmin(M, fmax(tp, (double)before(b))), m1 = fmin(M, (double)S.tot[b]);
    const int t0 = first_bin(S.tot, fmax(1.0, u * m0), S), t1 = first_bin(S.tot, fmax(1.0, u * m1), S);
    ok = t1 + 1 >= b ? gather(t0, b, 0, -1) : gather(t0, t1, b, b);
    if (ok) {
      reach(tp);
      M = fmin(M, (double)S.value);
      i = reach(fmax(1.0, u * M));
    } else {
      ok = gather(b, b, 0, -1);
      if (ok) {
        reach(tp);
        M = fmin(M, (double)S.value);
      }
    }
  }
  if (ok && i < 0) {
    const double target = fmax(1.0, u * M);
    const int b = first_bin(S.tot, target, S);
    ok = gather(b, b, 0, -1);
    if (ok) i = reach(target);
    ok = ok && i >= 0;
  }
  (void)command(Command{kExit, 0, 0, 0, 0});
  u64 c1;
  if (ok) {
    c1 = S.list[i];
  } else {
    c1 = draw_slowly(x, a.V, R, p, u, &M, S);
  }
  const float prob = (float)(exp(((double)Row::value(c1) - (double)top) * R.inv_t) * kUnit / M);
  finish((int64_t)(c1 & ((1u << kIdxBits) - 1)), prob);
}

size_t smem_bytes(int vchunk) { return ((sizeof(Shared) + 15) & ~size_t(15)) + (size_t)vchunk * 16; }

std::atomic<int> g_smem_set[3][kMaxDevicesAttr];
std::atomic<int> g_big_cluster[kMaxDevicesAttr];  // 0 unknown, 1 clusters of 8 at most, 2 of 16

}  // namespace

cudaError_t launch_draw(const DrawArgs& a, int sm_count, cudaStream_t st) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevicesAttr) return cudaErrorInvalidDevice;
  return with_type(a.ltype, [&](auto tv) -> cudaError_t {
    using T = decltype(tv);
    const void* fn = reinterpret_cast<const void*>(draw_kernel<T>);
    const int nvec = (a.V + 2 * (16 / (int)sizeof(T)) - 2) / (16 / (int)sizeof(T));  // with any lead
    // As many CTAs per row as leave two of them room on an SM; more for a few
    // rows, down to 128 vectors each
    int C = (int)(((size_t)nvec * 16 + kSliceBytes - 1) / kSliceBytes);
    const int spread = std::min(sm_count / std::max(1, a.rows), nvec / 128);
    C = std::max(1, std::min(std::max(C, spread), kMaxCluster));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.stream = st;
    cudaError_t e = cudaSuccess;
    auto shape = [&] {
      attr[0].val.clusterDim.x = (unsigned)C;
      cfg.gridDim = dim3((unsigned)(a.rows * C), 1, 1);
      cfg.dynamicSmemBytes = smem_bytes((nvec + C - 1) / C);
      e = ensure_smem_attr(fn, (int)cfg.dynamicSmemBytes, g_smem_set[sizeof(T) == 4 ? 0 : a.ltype]);
    };
    if (C > 8) {
      int known = g_big_cluster[dev].load(std::memory_order_relaxed);
      if (!known) {
        int n = 0;
        const int keep = C;
        C = kMaxCluster;
        e = cudaFuncSetAttribute(reinterpret_cast<const void*>(draw_kernel<float>),
                                 cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess)
          e = cudaFuncSetAttribute(reinterpret_cast<const void*>(draw_kernel<__half>),
                                   cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess)
          e = cudaFuncSetAttribute(reinterpret_cast<const void*>(draw_kernel<__nv_bfloat16>),
                                   cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) shape();
        known = e == cudaSuccess && cudaOccupancyMaxActiveClusters(&n, fn, &cfg) == cudaSuccess && n >= 1 ? 2 : 1;
        (void)cudaGetLastError();
        g_big_cluster[dev].store(known, std::memory_order_relaxed);
        C = keep;
      }
      if (known != 2) C = 8;
    }
    shape();
    if (e != cudaSuccess) return e;
    return cudaLaunchKernelEx(&cfg, draw_kernel<T>, a, (nvec + C - 1) / C);
  });
}

}  // namespace nls
