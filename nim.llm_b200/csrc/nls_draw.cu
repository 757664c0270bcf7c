// nls_draw.cu -- nls_draw_batch: one token per row from fp32, fp16 or bfloat16
// logits by temperature, top-k, top-p, min-p and a given uniform.
//
// The row's order is descending logits, equal ones by ascending index: token i
// has the place of comp(i) = (complement of the logit's ordered key, i), a
// 50-bit number. Every step of the definition keeps a prefix of that order, so
// a row needs no sort: only the tokens near the borders of its prefixes do.
// Masses are exp((x - max) / T) in fp64 (a table of 512 powers of two and a
// polynomial of degree 3, after Tang, ACM TOMS 15(2), 1989; within 2^-46 of the
// value), rounded to multiples of 2^-45 as they are summed: at most 2^18 of them
// stay below 2^63, and the sums are whole numbers, so their order does not
// matter (but for a mass half way between two multiples, which may go to
// either: 2^-45 of the largest).
//
// Where a row runs: with many rows, one CTA per row (four to an SM), which
// streams the row from memory; with few, a thread-block cluster per row, each
// CTA with its slice of the row in shared memory. Then one of two ways:
//  * Few candidates (top-k up to half the CTA's threads; min-p alone): a cut that at
//    least the needed tokens reach -- for top-k a quantile of the threads' maxima,
//    since the k-th largest of some of the logits is no larger than the k-th
//    largest of all -- and the tokens above it, collected and sorted by the
//    (first) CTA. A streamed row takes the cut from its first logits and reads
//    the row once.
//  * Masses of the whole row (no top-k, or the candidates were too many): the
//    masses of 1024 bins over the row's span of logits, to about 2^-13, say where
//    the border of each prefix and the token drawn lie. One pass then sums the
//    exact masses of the row and of what comes before those places, and collects
//    the tokens there, which are sorted. (A token adds its mass relative to its
//    bin's middle, by a polynomial of degree two in fp32, with one atomic.
//    Binning the exact masses instead took 35 more instructions per logit and
//    two returning atomics.) What the sums do not confirm, and bins at a border
//    that hold too many tokens (from about a thousand equal logits on), goes to a
//    radix selection over comp, ten bits at a time, by the (first) CTA: 1.5 to 2
//    ms a row of 150000 logits, and up to 35 ms where nearly all of them have one
//    of two or three values, whose additions meet at one address.
// What bounds it: reading the logits for the first way; for the second the
// instructions of the masses (about 40 per logit, 11 of them fp64, in the exact
// pass); for a few rows the chain of barriers of one row. Measured: 256 x 128256
// fp32, highest logit 29 us (4.5 TB/s), top-k 50 42 us, nucleus 161 us, settings
// of every kind 112 us; 2048 x 151936 bfloat16 top-k 50 248 us (2.5 TB/s); 64 x
// 151936 bfloat16 nucleus 75 us; one row of 128256: top-k with top-p and min-p
// 19 us, nucleus 36 us.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "nls_common.cuh"
#include "nls_kernels.h"
#include "nls_types.cuh"

namespace nls {

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxCluster = 16;
constexpr int kBins = 1024;
constexpr int kIdxBits = 18;
constexpr int kList = 2048;           // tokens the first CTA collects and sorts
constexpr int kMine = 1024;           // tokens a CTA hands over together
constexpr double kUnit = 35184372088832.0;  // 2^45
constexpr int kMaxWarps = 32;
constexpr int kPow2 = 512;            // the exponential's table

using u64 = unsigned long long;

// What the first CTA tells the others.
struct Command {
  int op;  // kExit, kMasses or kSums
  // kSums: the masses of logits >= ra and >= qa (before the two ranges), the
  // tokens from there down to rb and qb, the mass of logits >= enough
  float ra, rb, qa, qb, enough;
};
constexpr int kExit = 0, kMasses = 1, kSums = 2;
struct Sums {
  u64 all, enough;  // of the row; of its tokens with at least min_p
  u64 before_r, before_q;
};

struct Shared {
  u64 list[kList];
  union {
    // this CTA's bins: masses in 2^-13 of the middle's, and counts (for top-k)
    uint32_t bins[2][kBins];
    u64 mine[kMine];  // its tokens for the list
  };
  // (first CTA) running counts of the row's bins (of masses in 2^-13 before
  // that), and running masses by estimate
  uint32_t tcnt[kBins], tmass[kBins];
  union {
    double est[kBins];
    u64 tot[kBins];       // radix selection
  };
  double pow2[kPow2];  // 2^(j / 512)
  u64 red[kMaxWarps], reds[4][kMaxWarps];
  u64 first[kMaxCluster];  // each CTA's first highest logit
  Sums sums[kMaxCluster];
  float top[kMaxCluster], low[kMaxCluster];
  float fred[2][kMaxWarps];
  Command cmd;
  float ends[5];
  unsigned n_list, n_mine;
  int pick, picks[3];
  u64 value;
  u64 lo;              // radix selection
  u64 before;
};

// The exponential's constants (read as operands from constant memory: as
// immediates each would be moved to two registers for every logit): ln 2 / 512
// as l, l^2 / 2, l^3 / 6; 1.5 2^52.
constexpr double kL = 0.0013538030870311431;
__constant__ double kMassC[4] = {kL, kL * kL / 2.0, kL * kL * kL / 6.0, 6755399441055744.0};

// A row's largest logit and temperature, and the arithmetic of its masses.
struct Row {
  double top;          // the largest logit
  double scale;        // 512 / (T ln 2)
  float floor;         // logits below have no mass, -inf among them
  const double* pow2;
  __device__ __forceinline__ Row(float mx, double T, const double* table) : top((double)mx), pow2(table) {
    scale = __dmul_rn(fmin(1.0 / T, 1e300), 738.65986093514925);
    // e^-32.2 is less than half a unit (0.37 of one), and a logit below the float
    // nearest to max - 32.2 T lies below that itself
    floor = fmaxf((float)__dsub_rn(top, __dmul_rn(32.2, T)), -3.402823466e38f);
  }
  static __device__ __forceinline__ u64 comp(float v, int i) { return ((u64)(~fkey(v)) << kIdxBits) | (u64)i; }
  static __device__ __forceinline__ float value(u64 c) { return fkey_inv(~(uint32_t)(c >> kIdxBits)); }
  __device__ __forceinline__ bool has_mass(float v) const { return v >= floor; }
  // exp((v - max) / T) = 2^(n / 512) e^(f ln 2 / 512), n whole, |f| <= 1/2, of a
  // logit that has mass
  __device__ __forceinline__ double mass(float v) const {
    const double d = __dsub_rn((double)v, top);
    const double kd = __fma_rn(d, scale, kMassC[3]);  // + 1.5 2^52: rounded to n
    const int n = __double2loint(kd);
    const double f = __fma_rn(d, scale, -__dsub_rn(kd, kMassC[3]));
    const double p = __fma_rn(f, __fma_rn(f, kMassC[2], kMassC[1]), kMassC[0]);
    const double t = pow2[n & (kPow2 - 1)];
    // n / 512 into the exponent: bits 9 and up of n belong at bit 20
    const double s = __hiloint2double(__double2hiint(t) + ((n & ~(kPow2 - 1)) << 11), __double2loint(t));
    return __fma_rn(s, __dmul_rn(f, p), s);
  }
  // in units of 2^-45: the low bits beside 1.5 2^7, whose last place they are
  static __device__ __forceinline__ u64 units(double m) {
    return (u64)(__double_as_longlong(__dadd_rn(m, 192.0)) - __double_as_longlong(192.0));
  }
  __device__ __forceinline__ u64 units_of(float v) const { return has_mass(v) ? units(mass(v)) : 0ull; }
};

// acc += m where v >= from (as one predicated addition)
__device__ __forceinline__ void add_if(double& acc, double m, float v, float from) {
  asm("{\n\t.reg .pred p;\n\t"
      "setp.ge.f32 p, %2, %3;\n\t"
      "@p add.rn.f64 %0, %0, %1;\n\t}"
      : "+d"(acc)
      : "d"(m), "f"(v), "f"(from));
}

template <int NT>
__device__ u64 block_sum(u64 v, Shared& S) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) S.red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) t += S.red[w];
  return t;
}

// the running sum of v over the threads before this one
template <int NT>
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
  for (int w = 0; w < NT / 32; ++w)
    if (w < (int)(threadIdx.x >> 5)) t += S.red[w];
  return t;
}

// the first bin whose running sum reaches target, or -1
template <int NT, class V>
__device__ int first_bin(const V* run, double target, Shared& S) {
  __syncthreads();
  if (threadIdx.x == 0) S.pick = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += NT)
    if ((double)run[b] >= target && (b == 0 || (double)run[b - 1] < target)) S.pick = b;
  __syncthreads();
  return S.pick;
}

// first_bin of three targets
template <int NT>
__device__ void first_bins(const double* run, const double (&target)[3], int (&bin)[3], Shared& S) {
  __syncthreads();
  if (threadIdx.x < 3) S.picks[threadIdx.x] = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += NT) {
    const double at = run[b], before = b > 0 ? run[b - 1] : -1.0;
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (at >= target[k] && (b == 0 || before < target[k])) S.picks[k] = b;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) bin[k] = S.picks[k];
}

// S.list[0 .. n) ascending (n <= kList). Short lists by counting: four lanes find
// a token's place (all differ). Longer ones bitonic: a warp keeps 64 neighbours in
// registers for the strides below 64; larger strides go through shared memory,
// two at a time. (Few barriers: with one stride each, 555 tokens took 17000
// cycles.)
template <int NT>
__device__ void sort_list(int n, Shared& S) {
  const int lane = threadIdx.x & 31;
  if (n <= NT / 4) {
    const int i = threadIdx.x >> 2;
    __syncthreads();
    const u64 x = S.list[min(i, n)];
    int place = 0;
#pragma unroll 4
    for (int j = threadIdx.x & 3; j < n; j += 4) place += S.list[j] < x ? 1 : 0;
    place += __shfl_xor_sync(0xffffffffu, place, 1);
    place += __shfl_xor_sync(0xffffffffu, place, 2);
    __syncthreads();
    if (i < n && (threadIdx.x & 3) == 0) S.list[place] = x;
    __syncthreads();
    return;
  }
  int p = 64;
  while (p < n) p <<= 1;
  for (int i = n + (int)threadIdx.x; i < p; i += NT) S.list[i] = ~0ull;
  __syncthreads();
  auto order = [](u64& x, u64& y, bool up) {
    if ((x > y) == up) {
      const u64 t = x;
      x = y;
      y = t;
    }
  };
  auto in_warp = [&](u64& x, int stride, bool up) {
    const u64 y = __shfl_xor_sync(0xffffffffu, x, stride);
    if ((up == ((lane & stride) == 0)) ? y < x : y > x) x = y;
  };
  for (int size = 64; size <= p; size <<= 1) {
    int stride = size >> 1;
    if (size > 64) {
      if ((__ffs(size) & 1) == 0) {  // an odd number of strides above 32: one alone
        for (int i = threadIdx.x; i < p / 2; i += NT) {
          const int a = ((i & ~(stride - 1)) << 1) | (i & (stride - 1));
          u64 x = S.list[a], y = S.list[a + stride];
          order(x, y, (a & size) == 0);
          S.list[a] = x;
          S.list[a + stride] = y;
        }
        __syncthreads();
        stride >>= 1;
      }
      for (; stride > 32; stride >>= 2) {
        const int half = stride >> 1;
        for (int i = threadIdx.x; i < p / 4; i += NT) {
          const int a = ((i & ~(half - 1)) << 2) | (i & (half - 1));
          const bool up = (a & size) == 0;
          u64 w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = S.list[a + k * half];
          order(w[0], w[2], up);
          order(w[1], w[3], up);
          order(w[0], w[1], up);
          order(w[2], w[3], up);
#pragma unroll
          for (int k = 0; k < 4; ++k) S.list[a + k * half] = w[k];
        }
        __syncthreads();
      }
    }
    for (int base = 64 * (int)(threadIdx.x >> 5); base < p; base += 2 * NT) {
      u64 x = S.list[base + lane], y = S.list[base + 32 + lane];
      if (size == 64) {
#pragma unroll
        for (int z = 2; z <= 32; z <<= 1)
#pragma unroll
          for (int t = z >> 1; t > 0; t >>= 1) {
            in_warp(x, t, (lane & z) == 0);
            in_warp(y, t, z < 32 && (lane & z) == 0);
          }
      }
      const bool up = (base & size) == 0;
      order(x, y, up);
#pragma unroll
      for (int t = 16; t > 0; t >>= 1) {
        in_warp(x, t, up);
        in_warp(y, t, up);
      }
      S.list[base + lane] = x;
      S.list[base + 32 + lane] = y;
    }
    __syncthreads();
  }
}

// Radix selection over the whole row in memory: the smallest comp whose running
// count (by_count) or mass reaches target.
template <int NT, class T>
__device__ u64 select(const T* x, int V, const Row& R, bool by_count, double target, Shared& S) {
  if (target < 1.0) target = 1.0;
  if (threadIdx.x == 0) {
    S.lo = 0;
    S.before = 0;
  }
  for (int shift = 40; shift >= 0; shift -= 10) {
    for (int i = threadIdx.x; i < kBins; i += NT) S.tot[i] = 0;
    __syncthreads();
    const u64 lo = S.lo, before = S.before;
    for (int i0 = 0; i0 < V; i0 += NT) {
      const int i = i0 + (int)threadIdx.x;
      unsigned bin = kBins;  // (none)
      u64 w = 0;
      if (i < V) {
        const float v = to_f32(x[i]);
        const u64 d = Row::comp(v, i) - lo;
        if ((d >> (shift + 10)) == 0) {
          bin = (unsigned)(d >> shift);
          w = by_count ? 1ull : R.units_of(v);
        }
      }
      // A warp that meets one bin, as with equal logits, adds once: 64-bit
      // additions of every lane to one address took 34 ms for a row of 150000 equal
      // logits, which takes 1.5 ms so (rows of few equal ones 5 to 10 % more).
      if (__all_sync(0xffffffffu, bin == __shfl_sync(0xffffffffu, bin, 0))) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        if ((threadIdx.x & 31) != 0) w = 0;
      }
      if (w) atomicAdd(&S.tot[bin], w);
    }
    __syncthreads();
    constexpr int kPer = kBins / NT;
    const int b0 = kPer * threadIdx.x;
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += S.tot[b0 + i];
    u64 e = before + block_scan<NT>(sum, S);
    __syncthreads();
    if (threadIdx.x == 0) S.pick = -1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const u64 f = e + S.tot[b0 + i];
      if ((double)e < target && (double)f >= target) {
        S.pick = b0 + i;
        S.before = e;
      }
      e = f;
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
template <int NT, class T>
__device__ u64 draw_slowly(const T* x, int V, const Row& R, const nls_draw_params& p, double u, double* kept, Shared& S) {
  u64 bound = ~0ull;  // what is kept: comp <= bound
  if (p.top_k > 0 && p.top_k < V) bound = select<NT>(x, V, R, true, (double)p.top_k, S);
  if (p.top_p > 0.0 && p.top_p < 1.0) {
    u64 t = 0;
    for (int i = threadIdx.x; i < V; i += NT) {
      const float v = to_f32(x[i]);
      if (Row::comp(v, i) <= bound) t += R.units_of(v);
    }
    const u64 c = select<NT>(x, V, R, false, p.top_p * (double)block_sum<NT>(t, S), S);
    if (c < bound) bound = c;
  }
  u64 t = 0;
  for (int i = threadIdx.x; i < V; i += NT) {
    const float v = to_f32(x[i]);
    if (R.has_mass(v) && Row::comp(v, i) <= bound) {
      const double m = R.mass(v);
      if (!(p.min_p > 0.0 && m < p.min_p)) t += Row::units(m);
    }
  }
  *kept = (double)block_sum<NT>(t, S);
  return select<NT>(x, V, R, false, u * *kept, S);
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

// the larger of two, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// the largest of a vector, NaN if it holds one
template <class T>
__device__ __forceinline__ float vec_max(const uint4& q) {
  if constexpr (sizeof(T) == 4) {
    return max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)),
                   max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* h = reinterpret_cast<const T2*>(&q);
    const T2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(to_f32(m.x), to_f32(m.y));
  }
}

// NT threads. STREAM: one CTA per row, the row read from memory on each pass;
// else a cluster per row with vchunk 16-byte vectors of it per CTA.
template <class T, int NT, bool STREAM>
__global__ void __launch_bounds__(NT, STREAM ? 1024 / NT : 1) draw_kernel(const DrawArgs a, int vchunk) {
  constexpr int VN = Vec<T>::N, kWarps = NT / 32;
  constexpr int kPerBin = kBins / NT, kPerList = kList / NT;
  static_assert(kPerBin >= 1, "threads");
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& S = *reinterpret_cast<Shared*>(smem);
  uint4* slice = reinterpret_cast<uint4*>(smem + ((sizeof(Shared) + 15) & ~size_t(15)));
  const cg::cluster_group cluster = cg::this_cluster();
  const int C = STREAM ? 1 : (int)cluster.num_blocks(), rank = STREAM ? 0 : (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // few candidates: top-k up to half the threads (the quantile of their maxima
  // is near the k-th largest then), or min-p alone
  auto kind_of = [&](const nls_draw_params& p) {  // 0: highest logit, 1: few candidates, 2: masses
    if (p.temperature <= 0.0 || p.min_p > 1.0) return 0;
    const bool by_k = p.top_k > 0 && p.top_k < a.V;
    return by_k ? (p.top_k <= NT / 2 ? 1 : 2) : !(p.top_p > 0.0 && p.top_p < 1.0) && p.min_p > 0.0 ? 1 : 2;
  };
  int row = (int)(blockIdx.x / (unsigned)C);
  if constexpr (STREAM) {
    // Rows that need masses take about three times as long: they come first, so
    // that they start at once and each on an SM of its own.
    if (a.rows <= NT) {
      const bool mine = tid < a.rows && kind_of(a.params[tid]) == 2;
      const unsigned in_warp = __ballot_sync(0xffffffffu, mine);
      if (lane == 0) S.red[warp] = (u64)__popc(in_warp);
      __syncthreads();
      int at = __popc(in_warp & ((1u << lane) - 1u)), all = 0;  // such rows before this one; of all
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        all += (int)S.red[w];
        if (w < warp) at += (int)S.red[w];
      }
      if (tid < a.rows && (mine ? at : all + tid - at) == row) S.pick = tid;
      __syncthreads();
      row = S.pick;
    }
  }
  auto remote = [&](int r) -> Shared& { return STREAM ? S : *cluster.map_shared_rank(&S, r); };
  auto sync_all = [&] {
    if constexpr (STREAM) __syncthreads();
    else cluster.sync();
  };

  if (tid == 0) S.n_list = S.n_mine = 0;
  for (int i = tid; i < kPow2; i += NT) S.pow2[i] = exp2((double)i / kPow2);
  if constexpr (STREAM) __syncthreads();
  else asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const nls_draw_params p = a.params[row];
  const double u = a.uniforms ? a.uniforms[row] : -1.0;
  const bool by_k = p.top_k > 0 && p.top_k < a.V, by_p = p.top_p > 0.0 && p.top_p < 1.0, by_m = p.min_p > 0.0;
  const bool greedy = kind_of(p) == 0, few = kind_of(p) == 1;
  const bool masses = !greedy && !few;

  // The row, or the CTA's slice: vectors [v0, v0 + nv), counted from the 16-byte
  // boundary at or before the first logit. Vectors that reach past the row's
  // ends are read by element; what is not the row's is -inf, which is never
  // drawn and has no mass.
  const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.ld;
  const int lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int nvec = (lead + a.V + VN - 1) / VN;
  const int v0 = STREAM ? 0 : rank * vchunk, nv = STREAM ? nvec : max(0, min(vchunk, nvec - v0));
  const uint4* xv = reinterpret_cast<const uint4*>(x - lead) + v0;
  // whole vectors: [whole0, whole0 + whole_n)
  const int whole0 = v0 == 0 && lead > 0 ? 1 : 0;
  const uint32_t whole_n = (uint32_t)max(0, min(nv, (lead + a.V) / VN - v0) - whole0);
  auto load = [&](int i) -> uint4 {
    if ((uint32_t)(i - whole0) < whole_n) return __ldg(xv + i);
    const int first = (v0 + i) * VN - lead;  // the vector's first logit
    union {
      T e[VN];
      uint4 v;
    } w;
#pragma unroll
    for (int k = 0; k < VN; ++k)
      w.e[k] = i < nv && first + k >= 0 && first + k < a.V ? x[first + k] : from_f32<T>(-INFINITY);
    return w.v;
  };
  // f(i, vector i) for this thread's vectors, a whole warp together (i >= nv:
  // -inf throughout)
  constexpr int U = 16 / VN;  // loads per thread and batch (another batch is in flight)
  auto vectors = [&](auto&& f) {
    if constexpr (STREAM) {
      uint4 q[U], nx[U];
#pragma unroll
      for (int t = 0; t < U; ++t) q[t] = load(tid + t * NT);
      for (int j = tid; j - lane < nv; j += U * NT) {
        if (j - lane + U * NT < nv) {
#pragma unroll
          for (int t = 0; t < U; ++t) nx[t] = load(j + (U + t) * NT);
        }
#pragma unroll
        for (int t = 0; t < U; ++t) {
          f(j + t * NT, q[t]);
          q[t] = nx[t];
        }
      }
    } else {
      for (int j = tid; j - lane < nv; j += NT) f(j, j < nv ? slice[j] : load(nv));
    }
  };

  // The largest logit, and (for masses) the smallest of the first ones that have a
  // mass beside it: what is masked, by -inf or by a finite value, is not in the
  // span of the bins. (-1e9 on one logit made that span 32.5 T, its bins too full
  // to collect, and 64 x 151936 bfloat16 nucleus rows 1700 us instead of 80.)
  float top = -INFINITY, low = -INFINITY, cut = -INFINITY;
  const float depth = fminf((float)(32.2 * p.temperature), 3.402823466e38f);
  // the low of a part of the row whose largest logit is t, beside the largest of
  // more of it
  auto low_beside = [&](float t, float l, float largest) {
    const float f = largest - depth;
    return t >= f && t > -INFINITY ? fmaxf(l, f) : INFINITY;
  };
  // top and low of n parts, a lane each (the same in every lane afterwards)
  auto join = [&](const float* t, const float* l, int n) {
    const float mine = lane < n ? t[lane] : -INFINITY;
    top = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!masses) return;
    low = low_beside(mine, lane < n ? l[lane] : INFINITY, top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  };
  int best = 0;  // the first vector that holds this thread's largest logit
  // A cut that at least k of the block's values v (one per thread) reach, and
  // not many more: every warp's j-th largest, j = ceil(k / warps) (descending
  // sort of 32; the first `warps` warps have values throughout), the smallest of
  // those, then bisection between it and the largest.
  auto quantile = [&](float v, int k, int warps) -> float {
    float m = v;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
      for (int stride = size >> 1; stride > 0; stride >>= 1) {
        const float y = __shfl_xor_sync(0xffffffffu, m, stride);
        m = ((lane & size) == 0) == ((lane & stride) == 0) ? fmaxf(m, y) : fminf(m, y);
      }
    const int j = warps > 0 ? (k + warps - 1) / warps : 33;
    const float mj = __shfl_sync(0xffffffffu, m, min(j, 32) - 1);
    __syncthreads();
    if (lane == 0) {
      S.fred[0][warp] = mj;
      S.fred[1][warp] = m;
    }
    __syncthreads();
    float c = INFINITY, d = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warps) c = fminf(c, S.fred[0][w]);
      d = fmaxf(d, S.fred[1][w]);
    }
    if (j > 32 || !(c > -INFINITY) || !(d < INFINITY)) return -INFINITY;
    for (int i = 0; i < 8; ++i) {
      const float mid = 0.5f * c + 0.5f * d;
      if (!(mid > c && mid < d)) break;
      const int reached = __syncthreads_count(v >= mid);
      if (reached >= k) c = mid;
      else d = mid;
      if (reached >= k && reached <= k + k / 8) break;
    }
    return c;
  };
  // The cut of what this CTA has seen so far: of the threads' maxima for top-k;
  // or a little below max + T ln(min_p) (the masses decide).
  auto find_cut = [&] {
    if (by_k) {
      cut = quantile(top, (int)p.top_k, min(kWarps, nv / 32));
    } else {
      float m = top;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      __syncthreads();
      if (lane == 0) S.fred[0][warp] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, S.fred[0][w]);
      const float f = (float)((double)m + p.temperature * log(p.min_p));
      cut = f == f ? f - fmaxf(fabsf(f), fabsf(m)) * 0x1p-20f : -INFINITY;
    }
  };
  // A token's bin: its distance below `ref` in 1023rds of the span, rounded to a
  // whole number by adding 2^23 (those below the span are in the last bin; the
  // span reaches at least to the smallest of the first logits or to max - 32.5 T,
  // below which nothing has a mass). The span is finite and not negative,
  // whatever the temperature, and where the first logits seen are all -inf (`to`
  // is +inf then).
  float ref = 0.0f, span = 0.0f, scale = 0.0f, floor = 0.0f, c1 = 0.0f, c2 = 0.0f;
  constexpr float kWhole = 8388608.0f;  // 2^23
  auto bin_of = [](float b) { return (int)min(__float_as_uint(b) - 0x4B000000u, (uint32_t)(kBins - 1)); };
  auto bin = [&](float v) { return bin_of(__fmaf_rn(fminf(ref - v, span), scale, kWhole)); };
  // from, to: the span; seen: the largest logit so far (what has no mass beside it
  // has none beside a larger one)
  auto set_bins = [&](float from, float to, float seen) {
    const float above = fmaxf(from - seen, 0.0f);
    const float widest = fminf((float)(32.5 * p.temperature) + above, 3.402823466e38f);
    ref = from;
    span = to <= from ? fminf(from - to, widest) : widest;
    scale = span > 1e-30f ? (float)(kBins - 1) / span : 0.0f;
    const double step = scale > 0.0f ? -1.0 / ((double)scale * p.temperature) : 0.0;
    // 2^13 e^(step f) = 2^13 (1 + step f + (step f)^2 / 2), f the distance from
    // the bin's middle in bins
    c1 = (float)(8192.0 * step);
    c2 = (float)(4096.0 * step * step);
    floor = Row(seen, p.temperature, nullptr).floor;
  };
  auto add_bins = [&](const uint4& q) {
    if (!(vec_max<T>(q) >= floor)) return;
    const Vec<T> e(q);
#pragma unroll
    for (int k = 0; k < VN; ++k) {
      const float d = fminf(ref - e.v[k], span), b = __fmaf_rn(d, scale, kWhole);
      const float f = __fmaf_rn(d, scale, kWhole - b);
      const float w = __fmaf_rn(f, __fmaf_rn(f, c2, c1), kWhole + 8192.0f);  // (the low bits beside 2^23)
      const int i = bin_of(b);
      if (e.v[k] >= floor) {
        atomicAdd(&S.bins[0][i], __float_as_uint(w) - 0x4B000000u);
        if (by_k) atomicAdd(&S.bins[1][i], 1u);
      }
    }
  };
  // A streamed row's first pass fills the bins too, from the largest of its first
  // logits and a quarter of their span above; a larger one makes a pass of its
  // own necessary.
  const bool binned = STREAM && masses && p.temperature > 0.0;
  {
    constexpr int U = 4;
    uint4 q[U], nx[U];
#pragma unroll
    for (int t = 0; t < U; ++t) q[t] = load(tid + t * NT);
    for (int j0 = 0, batch = 0; j0 < nv; j0 += U * NT, ++batch) {
      if (j0 + U * NT < nv) {
#pragma unroll
        for (int t = 0; t < U; ++t) nx[t] = load(tid + j0 + (U + t) * NT);
      }
      float vm[U];
#pragma unroll
      for (int t = 0; t < U; ++t) {
        const int i = tid + j0 + t * NT;
        if (!STREAM && i < nv) slice[i] = q[t];
        vm[t] = vec_max<T>(q[t]);
        if (STREAM && vm[t] > top) best = i;
        top = max_nan(top, vm[t]);
      }
      // (the span of the bins need not be the whole row's: a thread looks at its
      // first logits, and again where all so far have no mass beside a new one)
      if (masses && !(low >= top - depth)) {
        const float f = top - depth;
        low = INFINITY;
#pragma unroll
        for (int t = 0; t < U; ++t) {
          const Vec<T> e(q[t]);
#pragma unroll
          for (int k = 0; k < VN; ++k) low = fminf(low, e.v[k] >= f ? e.v[k] : INFINITY);
        }
      }
      if (STREAM && binned) {
        if (batch == 0) {
          float m = top;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          float l = low_beside(top, low, m);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) l = fminf(l, __shfl_xor_sync(0xffffffffu, l, o));
          if (lane == 0) {
            S.fred[0][warp] = m;
            S.fred[1][warp] = l;
          }
          for (int i = tid; i < kBins; i += NT) S.bins[0][i] = S.bins[1][i] = 0;
          __syncthreads();
          const float mw = lane < kWarps ? S.fred[0][lane] : -INFINITY;
          m = mw;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          l = low_beside(mw, lane < kWarps ? S.fred[1][lane] : INFINITY, m);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) l = fminf(l, __shfl_xor_sync(0xffffffffu, l, o));
          m = fmaxf(m, -3.402823466e38f);
          set_bins(fminf(m + 0.25f * fminf(m - fminf(l, m), (float)(32.5 * p.temperature)), 3.402823466e38f), l, m);
        }
#pragma unroll
        for (int t = 0; t < U; ++t) add_bins(q[t]);
      }
      if (STREAM && few) {
        // the cut rises as more of the row has been seen
        if (batch == 0 || batch == 3 || batch == 15 || batch == 63) find_cut();
#pragma unroll
        for (int t = 0; t < U; ++t) {
          if (vm[t] >= cut && vm[t] > -INFINITY) {
            const Vec<T> e(q[t]);
            const int first = (tid + j0 + t * NT) * VN - lead;
#pragma unroll
            for (int k = 0; k < VN; ++k)
              if (e.v[k] >= cut && e.v[k] > -INFINITY) {
                const unsigned at = atomicAdd(&S.n_list, 1u);
                if (at < kList) S.list[at] = Row::comp(e.v[k], first + k);
              }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < U; ++t) q[t] = nx[t];
    }
  }
  if (!STREAM && few) find_cut();
  const float mine_top = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (masses) {
    low = low_beside(mine_top, low, top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  __syncthreads();
  if (lane == 0) {
    S.fred[0][warp] = top;
    S.fred[1][warp] = low;
  }
  __syncthreads();
  join(S.fred[0], S.fred[1], kWarps);
  if constexpr (!STREAM) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA has begun
    if (tid < C) {
      Shared& D = remote(tid);
      D.top[rank] = top;
      D.low[rank] = low;
    }
    cluster.sync();
    join(S.top, S.low, C);
  }

  int err = NLS_OK;
  if (!(fabsf(top) < INFINITY)) err = NLS_ERR_NAN_LOGITS;
  else if (!(p.temperature <= 0.0) && (!(p.temperature > 0.0) || !(u >= 0.0 && u < 1.0))) err = NLS_ERR_INVALID_ARG;
  auto finish = [&](int64_t id, float prob) {
    a.out_ids[row] = id;
    if (a.out_probs) a.out_probs[row] = prob;
  };
  if (err != NLS_OK) {  // (all CTAs agree; nothing remote is in flight)
    if (rank == 0 && tid == 0) {
      finish(-1, 0.0f);
      record_status(a.status, err);
    }
    return;
  }
  if (greedy) {
    // the first of the highest logits
    unsigned at = ~0u;
    if constexpr (STREAM) {
      if (mine_top == top) {
        const Vec<T> e(load(best));
#pragma unroll
        for (int k = VN - 1; k >= 0; --k)
          if (e.v[k] == top) at = (unsigned)(best * VN - lead + k);
      }
    } else {
      vectors([&](int i, const uint4& q) {
        const Vec<T> e(q);
#pragma unroll
        for (int k = 0; k < VN; ++k)
          if (i < nv && e.v[k] == top) at = min(at, (unsigned)((v0 + i) * VN - lead + k));
      });
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (tid == 0) S.value = ~0ull;
    __syncthreads();
    if (lane == 0) atomicMin(&S.value, (u64)at);
    __syncthreads();
    if (tid == 0) remote(0).first[rank] = S.value;
    sync_all();
    if (rank == 0 && tid == 0) {
      u64 m = ~0ull;
      for (int r = 0; r < C; ++r) m = min(m, S.first[r]);
      finish((int64_t)m, 1.0f);
    }
    return;
  }
  const Row R(top, p.temperature, S.pow2);

  // Tokens go to the (first) CTA's list (its count passes kList where they do
  // not all fit): one by one by each thread, then, from the CTAs' own lists, all
  // together. The latter ends with a barrier of all. What a CTA's own list has no
  // room for goes to the first CTA's at once: where most of a row is masked, the
  // tokens of one CTA may be all there are. (64 x 150001 bfloat16 nucleus rows with
  // the second half masked: 1100 us with those rows left to the selection over
  // the row, 80 so.)
  auto put = [&](float v, int i) {
    const unsigned at = atomicAdd(STREAM ? &S.n_list : &S.n_mine, 1u);
    if (STREAM) {
      if (at < kList) S.list[at] = Row::comp(v, i);
    } else if (at < kMine) {
      S.mine[at] = Row::comp(v, i);
    } else if (at < kList) {
      Shared& D = remote(0);
      const unsigned there = atomicAdd(&D.n_list, 1u);
      if (there < kList) D.list[there] = Row::comp(v, i);
    }
  };
  auto hand_over = [&] {
    __syncthreads();
    if constexpr (!STREAM) {
      const unsigned n = min(S.n_mine, (unsigned)kMine);
      Shared& D = remote(0);
      if (tid == 0) S.value = atomicAdd(&D.n_list, S.n_mine <= kList ? n : (unsigned)kList + 1u);
      __syncthreads();
      if (tid == 0) S.n_mine = 0;
      const unsigned at = (unsigned)S.value;
      if (at + n <= kList)
        for (unsigned i = tid; i < n; i += NT) D.list[at + i] = S.mine[i];
      cluster.sync();
    }
  };
  // the first CTA's next command (the others' arguments are ignored)
  auto command = [&](const Command& c) -> Command {
    if constexpr (STREAM) return c;
    if (rank == 0 && tid < C) remote(tid).cmd = c;
    cluster.sync();
    return S.cmd;
  };

  int n = 0;           // tokens in the list
  int per = 1;         // neighbours in it per thread (kPerList where they are more than threads)
  u64 run[kPerList];   // their running masses
  auto place = [&](int k) { return k < per ? per * tid + k : INT_MAX; };
  // the first of them whose running mass reaches target: its place in the
  // list (-1: none), and that mass in S.value
  auto reach = [&](double target) -> int {
    int at = INT_MAX;
#pragma unroll
    for (int k = kPerList - 1; k >= 0; --k)
      if (place(k) < n && (double)run[k] >= target) at = place(k);
    at = __reduce_min_sync(0xffffffffu, at);
    __syncthreads();
    if (tid == 0) S.pick = INT_MAX;
    __syncthreads();
    if (lane == 0 && at != INT_MAX) atomicMin(&S.pick, at);
    __syncthreads();
    const int i = S.pick;
    if (i == INT_MAX) return -1;
#pragma unroll
    for (int k = 0; k < kPerList; ++k)
      if (i == place(k)) S.value = run[k];
    __syncthreads();
    return i;
  };
  auto give = [&](u64 c, double M) {
    if (tid == 0)
      finish((int64_t)(c & ((1u << kIdxBits) - 1)),
             (float)(R.mass(Row::value(c)) * kUnit / M));
  };

  // ---- few candidates ---------------------------------------------------------
  if (few) {
    if constexpr (!STREAM) {
      vectors([&](int i, const uint4& q) {
        if (!(vec_max<T>(q) >= cut)) return;
        const Vec<T> e(q);
#pragma unroll
        for (int k = 0; k < VN; ++k)
          if (e.v[k] >= cut && e.v[k] > -INFINITY) put(e.v[k], (v0 + i) * VN - lead + k);
      });
      hand_over();
    }
    const unsigned found = S.n_list;
    const Command c = command(Command{found <= kList ? kExit : kMasses});
    if (c.op == kExit) {
      if (rank != 0) return;
      n = (int)found;
      if (by_k && n > 2 * (int)p.top_k && n >= NT / 4) {
        // most of the list is from cuts of less than the row: a cut of the list
        float m = -INFINITY;
        for (int i = tid; i < n; i += NT) m = fmaxf(m, Row::value(S.list[i]));
        const float c = quantile(m, (int)p.top_k, min(kWarps, n / 32));
        __syncthreads();
        for (int i = tid; i < n; i += NT) {
          const u64 v = S.list[i];
          if (Row::value(v) >= c) {
            const unsigned at = atomicAdd(&S.n_mine, 1u);
            if (at < kMine) S.mine[at] = v;
          }
        }
        __syncthreads();
        const int left = (int)S.n_mine;
        if (left <= kMine) {
          n = left;
          for (int i = tid; i < n; i += NT) S.list[i] = S.mine[i];
        }
        __syncthreads();
      }
      sort_list<NT>(n, S);
      if (by_k) n = min(n, (int)p.top_k);  // tokens kept by top-k
      per = n <= NT ? 1 : kPerList;
      u64 t = 0;
      unsigned enough = 0;  // which of them have at least min_p
#pragma unroll
      for (int k = 0; k < kPerList; ++k) {
        const float v = place(k) < n ? Row::value(S.list[place(k)]) : -INFINITY;
        const double m = R.has_mass(v) ? R.mass(v) : 0.0;
        if (!by_m || !(m < p.min_p)) enough |= 1u << k;
        t += Row::units(m);
        run[k] = t;
      }
      const u64 e = block_scan<NT>(t, S);
      __syncthreads();
      if (tid == NT - 1) S.value = e + t;
      __syncthreads();
      const double tp = by_p ? fmax(1.0, p.top_p * (double)S.value) : 0.0;
      // the kept mass: the last token's with what is before it short of top-p's
      // mass, and at least min_p itself
      u64 kept = 0, prev = e;
#pragma unroll
      for (int k = 0; k < kPerList; ++k) {
        run[k] += e;
        if (place(k) < n && (!by_p || (double)prev < tp) && (enough & (1u << k))) kept = run[k];
        prev = run[k];
      }
      __syncthreads();
      if (tid == 0) S.value = 0;
      __syncthreads();
      if (kept) atomicMax(&S.value, kept);
      __syncthreads();
      const double M = (double)S.value;
      const int i = reach(fmax(1.0, u * M));
      give(S.list[max(i, 0)], M);
      return;
    }
  }

  // ---- masses of the whole row ------------------------------------------------
  __syncthreads();
  if (few) {  // (its first pass took no low)
    const float f = top - depth;
    low = INFINITY;
    vectors([&](int, const uint4& q) {
      if (!(vec_max<T>(q) >= f)) return;
      const Vec<T> e(q);
#pragma unroll
      for (int k = 0; k < VN; ++k) low = fminf(low, e.v[k] >= f ? e.v[k] : INFINITY);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    if (lane == 0) S.fred[0][warp] = low;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) low = fminf(low, S.fred[0][w]);
    if constexpr (!STREAM) {
      if (tid < C) remote(tid).low[rank] = low;
      cluster.sync();
      for (int r = 0; r < C; ++r) low = fminf(low, S.low[r]);
    }
  }
  if (!binned || !(top <= ref)) {
    set_bins(top, low, top);
    for (int i = tid; i < kBins; i += NT) S.bins[0][i] = S.bins[1][i] = 0;
    __syncthreads();
    vectors([&](int, const uint4& q) { add_bins(q); });
  }
  // ln(mass) per bin, and the bins' zero from the largest logit
  const double step = scale > 0.0f ? -1.0 / ((double)scale * p.temperature) : 0.0;
  const double zero = ((double)ref - (double)top) / p.temperature;
  sync_all();
  // each CTA adds up its share of the bins
  {
    Shared& D = remote(0);
    const int b0 = kBins * rank / C, b1 = kBins * (rank + 1) / C;
    for (int b = b0 + tid; b < b1; b += NT) {
      uint32_t m = 0, k = 0;
      for (int r = 0; r < C; ++r) {
        m += remote(r).bins[0][b];
        if (by_k) k += remote(r).bins[1][b];
      }
      D.tmass[b] = m;
      D.tcnt[b] = by_k ? k : (m + 4096u) >> 13;  // (nearly, where no count has to be exact)
    }
  }
  sync_all();

  // The sums and tokens of a command, into the first CTA. Ends with a barrier
  // of all.
  auto add_up = [&](const Command& c) {
    Sums z{0, 0, 0, 0};
    const bool two = c.qb < c.qa;  // a second range
    __syncthreads();
    auto pass = [&](auto with_m, auto with_q) {
      vectors([&](int i, const uint4& q) {
        if (!__any_sync(0xffffffffu, R.has_mass(vec_max<T>(q)))) return;
        // four logits at a time (eight would not fit the registers); 192 = 1.5
        // 2^7: its last place is a unit, and their masses do not change its
        // exponent
#pragma unroll 1
        for (int g = 0; g < VN; g += 4) {
          float e[4];
          if constexpr (VN == 4) {
            e[0] = __uint_as_float(q.x);
            e[1] = __uint_as_float(q.y);
            e[2] = __uint_as_float(q.z);
            e[3] = __uint_as_float(q.w);
          } else {
            const Vec<T> both(g == 0 ? make_uint4(q.x, q.y, 0u, 0u) : make_uint4(q.z, q.w, 0u, 0u));
#pragma unroll
            for (int k = 0; k < 4; ++k) e[k] = both.v[k];
          }
          double all = 192.0, before_r = 192.0, before_q = 192.0, enough = 192.0;
          bool hit = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float v = e[k];
            const double m = R.mass(v);
            add_if(all, m, v, R.floor);
            add_if(before_r, m, v, c.ra);
            if (with_m.value) add_if(enough, m, v, c.enough);
            hit |= v >= c.rb && v < c.ra;
            if (with_q.value) {
              add_if(before_q, m, v, c.qa);
              hit |= v >= c.qb && v < c.qa;
            }
          }
          auto units = [](double x) { return (u64)(__double_as_longlong(x) - __double_as_longlong(192.0)); };
          z.all += units(all);
          z.before_r += units(before_r);
          if (with_m.value) z.enough += units(enough);
          if (with_q.value) z.before_q += units(before_q);
          if (hit) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float v = e[k];
              if ((v >= c.rb && v < c.ra) || (with_q.value && v >= c.qb && v < c.qa))
                put(v, (v0 + i) * VN - lead + g + k);
            }
          }
        }
      });
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (two) {
      if (by_m) pass(Yes{}, Yes{});
      else pass(No{}, Yes{});
    } else {
      if (by_m) pass(Yes{}, No{});
      else pass(No{}, No{});
    }
    hand_over();
    // the block's four sums, a warp each
    u64 v[4] = {z.all, z.enough, z.before_r, z.before_q};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
      if (lane == 0) S.reds[k][warp] = v[k];
    }
    __syncthreads();
    if (warp < 4) {
      u64 t = lane < kWarps ? S.reds[warp][lane] : 0ull;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      Sums& D = remote(0).sums[rank];
      if (lane == 0) (warp == 0 ? D.all : warp == 1 ? D.enough : warp == 2 ? D.before_r : D.before_q) = t;
    }
    sync_all();
  };
  if (rank != 0) {
    while (true) {
      const Command c = command(Command{});
      if (c.op == kExit) return;
      add_up(c);
    }
  }

  // running counts and masses of the bins
  {
    u64 k = 0;
    double m = 0.0, own[kPerBin];
#pragma unroll
    for (int i = 0; i < kPerBin; ++i) {
      const int b = kPerBin * tid + i;
      k += S.tcnt[b];
      own[i] = (double)S.tmass[b] * (exp(fmin(step * (double)b + zero, 40.0)) * 0x1p-13);
      m += own[i];
    }
    u64 f = block_scan<NT>(k, S);
    // (in 2^-40 of a largest mass: below 2^19 2^40)
    double e = (double)block_scan<NT>((u64)(m * 0x1p40), S) * 0x1p-40;
#pragma unroll
    for (int i = 0; i < kPerBin; ++i) {
      const int b = kPerBin * tid + i;
      S.tcnt[b] = (uint32_t)(f += S.tcnt[b]);
      S.est[b] = e += own[i];
    }
    __syncthreads();
  }
  // tokens of bins b0 .. b1 (nearly)
  auto held = [&](int b0, int b1) { return (int)(S.tcnt[b1] - (b0 > 0 ? S.tcnt[b0 - 1] : 0u)); };
  // The bins where a running mass of `lo` .. `hi`, `mid` most likely, may lie by
  // the estimates (a token's is off by its rounding, 2^-14, and what the
  // polynomial leaves, (step / 2)^3 / 6); no more of them than hold `most`
  // tokens, about the middle (many tokens' errors even out).
  const double wide = 1.0 + 0x1p-13 - step * step * step / 24.0;
  auto window = [&](double lo, double mid, double hi, int most, int* b0, int* b1) {
    const double total = S.est[kBins - 1];
    int at[3];
    first_bins<NT>(S.est, {fmin(lo / wide, total), fmin(mid, total), fmin(hi * wide, total)}, at, S);
    int l = max(at[0], 0), h = at[2] < 0 ? kBins - 1 : at[2];
    const int m = max(l, min(at[1] < 0 ? kBins - 1 : at[1], h));
    if (held(l, h) > most) {
      const int side = max(0, most - held(m, m)) / 2;
      const double below = (double)(m > 0 ? S.tcnt[m - 1] : 0u) - side, above = (double)S.tcnt[m] + side + 1.0;
      if (below > 0.0) l = max(l, first_bin<NT>(S.tcnt, below, S) + 1);
      const int x = first_bin<NT>(S.tcnt, above, S);
      if (x > 0) h = min(h, x - 1);
      l = min(l, m);
      h = max(h, m);
    }
    *b0 = l;
    *b1 = h;
  };
  // Sums and tokens of bins r0 .. r1 and q0 .. q1 (r1 < q0, or q1 < q0 for
  // none); run[] are the tokens' running masses in the row. False: too many.
  Sums z;
  int n_r = 0;
  auto look = [&](int r0, int r1, int q0, int q1) -> bool {
    __syncthreads();
    if (tid == 0) S.n_list = 0;
    __syncthreads();
    // The ranges as logits: the smallest of bin < r0, <= r1, < q0 and <= q1 (a bin
    // never rises with the logit), and the smallest with at least min_p; five
    // lanes, by bisection over the ordered keys.
    if (warp == 0) {
      const int most = lane == 0 ? r0 - 1 : lane == 1 ? r1 : lane == 2 ? q0 - 1 : q1;
      auto reached = [&](float v) { return lane < 4 ? bin(v) <= most : R.mass(v) >= p.min_p; };
      uint32_t under = fkey(R.floor) - 1u, upper = fkey(top);  // under: not reached (or no mass); upper: reached
      if (lane >= (by_m ? 5 : 4)) under = upper - 1u;  // (nothing to find)
      const bool any = lane < 4 ? bin(top) <= most : true;  // (else no logit is)
      while (__any_sync(0xffffffffu, upper - under > 1u)) {
        const uint32_t mid = under + (upper - under) / 2u;
        if (upper - under > 1u) {
          if (reached(fkey_inv(mid))) upper = mid;
          else under = mid;
        }
      }
      if (lane < 5) S.ends[lane] = any ? fkey_inv(upper) : INFINITY;
    }
    __syncthreads();
    const Command c = command(Command{kSums, S.ends[0], S.ends[1], q0 <= q1 ? S.ends[2] : INFINITY,
                                      q0 <= q1 ? S.ends[3] : INFINITY, S.ends[4]});
    add_up(c);
    n = (int)S.n_list;
    z = S.sums[0];
    for (int r = 1; r < C; ++r) {
      z.all += S.sums[r].all;
      z.enough += S.sums[r].enough;
      z.before_r += S.sums[r].before_r;
      z.before_q += S.sums[r].before_q;
    }
    if (n > kList) return false;
    sort_list<NT>(n, S);
    per = n <= NT ? 1 : kPerList;
    u64 t = 0, inside = 0;  // inside: the tokens of r0 .. r1, n_r of them
    int here = 0;
#pragma unroll
    for (int k = 0; k < kPerList; ++k) {
      if (place(k) < n) {
        const float v = Row::value(S.list[place(k)]);
        const u64 w = R.units_of(v);
        t += w;
        if (v >= c.rb) {
          inside += w;
          ++here;
        }
      }
      run[k] = t;
    }
    const u64 e = block_scan<NT>(t, S);
    if (q0 <= q1) {
      inside = block_sum<NT>(inside, S);
      n_r = (int)block_sum<NT>((u64)here, S);
    }
#pragma unroll
    for (int k = 0; k < kPerList; ++k) {
      const bool first = place(k) >= n || Row::value(S.list[place(k)]) >= c.rb;
      run[k] += e + (first ? z.before_r : z.before_q - inside);
    }
    return true;
  };

  bool ok = true;
  u64 total = 0;          // what top-k kept (or all)
  double total_est = S.est[kBins - 1];
  bool known = false;     // total is exact
  if (by_k) {
    // (no bin: all tokens with a mass are kept)
    const int b = first_bin<NT>(S.tcnt, (double)p.top_k, S);
    if (b >= 0) {
      ok = look(b, b, kBins, kBins - 1);
      if (ok) {
        // (past the bin's tokens: they are all kept as well, the border lies among
        // tokens without a mass, which the bins of a first pass may count)
        const int i = (int)(p.top_k - 1) - (b > 0 ? (int)S.tcnt[b - 1] : 0);
        __syncthreads();
        if (i >= n && tid == 0) S.value = z.all;
#pragma unroll
        for (int k = 0; k < kPerList; ++k)
          if (i == place(k) && i < n) S.value = run[k];
        __syncthreads();
        total = S.value;
        total_est = (double)total / kUnit;
        known = true;
      }
    }
  }
  int i = -1;
  double M = 0.0;
  if (ok) {
    // the kept mass by estimate, at least and at most; the bins of top-p's
    // border and of the drawn token
    double m = total_est, m0 = known ? m : m / wide, m1 = known ? m : m * wide;
    int q0 = kBins, q1 = kBins - 1, r0, r1;
    if (by_p) {
      m *= p.top_p;
      window(m0 * p.top_p, m, m1 * p.top_p, kList / 2 - 64, &q0, &q1);
      // (the token at the border is kept whole)
      m0 = fmax(m0 * p.top_p, q0 > 0 ? S.est[q0 - 1] / wide : 0.0);
      m1 = fmin(m1, S.est[q1] * wide);
    }
    if (by_m) {
      // the bin where min_p lies (two, next to a border: bin() is in fp32), and the
      // mass down to there; the first token is always kept
      const double lb = step < 0.0 ? fmax(0.0, fmin((log(p.min_p) - zero) / step, (double)kBins)) : (double)kBins;
      const int b = min(kBins - 1, (int)(lb + 0.49)), c = min(kBins - 1, (int)(lb + 0.51));
      const double before = b > 0 ? S.est[b - 1] : 0.0;
      m = fmin(m, fmax(1.0, before + (lb + 0.5 - (double)b) * (S.est[b] - before)));
      m1 = fmin(m1, S.est[c] * wide);
      m0 = fmin(m0, fmax(1.0, before / wide));
    }
    // (min-p alone leaves a bin's mass open, and the whole list to the bins that
    // may hold the token)
    window(u * m0, u * m, u * m1, by_m && !by_p ? kList - 64 : kList / 2 - 64, &r0, &r1);
    if (q0 <= q1 && r1 + 1 >= q0) {  // one range
      r0 = min(r0, q0);
      r1 = max(r1, q1);
      q0 = kBins;
      q1 = kBins - 1;
    }
    ok = look(r0, r1, q0, q1);
    if (ok) {
      if (!known) total = z.all;
      u64 kept = total;
      if (by_p) {
        // the border has to lie among the collected tokens of its bins
        const double tp = fmax(1.0, p.top_p * (double)total);
        const int at = reach(tp);
        const int skip = q0 <= q1 ? n_r : 0;
        ok = at >= skip && (double)(q0 <= q1 ? z.before_q : z.before_r) < tp;
        if (ok) kept = S.value < kept ? S.value : kept;
      }
      if (by_m && z.enough < kept) kept = z.enough;
      M = (double)kept;
      const double target = fmax(1.0, u * M);
      if (ok) {
        i = reach(target);
        // found among the tokens of r0 .. r1, or, in one range or the other,
        // right after what comes before it
        ok = i >= 0 && (double)z.before_r < target;
        if (ok && q0 <= q1 && i >= n_r) ok = (double)z.before_q < target;
      }
    }
  }
  (void)command(Command{kExit});
  const u64 drawn = ok ? S.list[i] : draw_slowly<NT>(x, a.V, R, p, u, &M, S);  // (sets M: before it is read)
  give(drawn, M);
}

constexpr int kMaxSmem = 227 * 1024;

size_t smem_bytes(int vchunk) { return ((sizeof(Shared) + 15) & ~size_t(15)) + (size_t)vchunk * 16; }

std::atomic<int> g_smem_set[4][3][kMaxDevicesAttr];
std::atomic<int> g_big_cluster[2][3][kMaxDevicesAttr];  // 0 unknown, 1 clusters of 8 at most, 2 of 16

}  // namespace

cudaError_t launch_draw(const DrawArgs& a, int sm_count, cudaStream_t st) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevicesAttr) return cudaErrorInvalidDevice;
  return with_type(a.ltype, [&](auto tv) -> cudaError_t {
    using T = decltype(tv);
    constexpr int VN = 16 / (int)sizeof(T);
    const int nvec = (a.V + 2 * VN - 2) / VN;  // with any lead
    cudaLaunchConfig_t cfg = {};
    cfg.stream = st;
    cudaError_t e = cudaSuccess;
    // CTAs per row: what shares the SMs among the rows, at least 128 vectors
    // each, at most 16 (8 where the device has no room for 16), and enough to
    // hold the row. Rows that would not all be on the device at once so are
    // streamed.
    const int most = (kMaxSmem - (int)smem_bytes(0)) / 16;
    const int need = (nvec + most - 1) / most;
    int C = std::min({sm_count / std::max(1, a.rows), nvec / 128, kMaxCluster});
    C = std::max({C, need, 1});
    if ((int64_t)C * a.rows > sm_count && nvec > 128) {
      // 1024 threads to an SM: four rows, or two where there are not that many
      // (256 x 128256 fp32 with 512 and with 1024 threads a row: top-k 42 and 53
      // us, nucleus 162 and 175, settings of every kind 113 and 99; 2048 x 151936
      // bfloat16 top-k with 256 and with 512 threads: 247 and 266 us, 500 x 50257
      // fp16 nucleus 149 and 158, 500 x 128256 fp32 of every kind 232 and 153: more
      // threads are better for the few rows that need masses, and which those are
      // is not known here)
      const bool many = a.rows > 3 * sm_count;
      auto stream = [&](auto kernel, int threads, std::atomic<int>* set) {
        cudaError_t f = ensure_smem_attr(reinterpret_cast<const void*>(kernel), (int)smem_bytes(0), set);
        if (f != cudaSuccess) return f;
        cfg.blockDim = dim3((unsigned)threads, 1, 1);
        cfg.gridDim = dim3((unsigned)a.rows, 1, 1);
        cfg.dynamicSmemBytes = smem_bytes(0);
        return cudaLaunchKernelEx(&cfg, kernel, a, 0);
      };
      return many ? stream(draw_kernel<T, 256, true>, 256, g_smem_set[2][a.ltype])
                  : stream(draw_kernel<T, 512, true>, 512, g_smem_set[3][a.ltype]);
    }
    // one CTA per SM at most: 1024 threads, or 256 where a CTA's share is less
    // than a vector for each of those
    const int wide = (nvec + C - 1) / C > 1024 ? 1 : 0;
    const auto kernel = wide ? draw_kernel<T, 1024, false> : draw_kernel<T, 256, false>;
    const void* fn = reinterpret_cast<const void*>(kernel);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(wide ? 1024u : 256u, 1, 1);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto shape = [&] {
      attr[0].val.clusterDim.x = (unsigned)C;
      cfg.gridDim = dim3((unsigned)(a.rows * C), 1, 1);
      cfg.dynamicSmemBytes = smem_bytes((nvec + C - 1) / C);
      e = ensure_smem_attr(fn, (int)cfg.dynamicSmemBytes, g_smem_set[wide][a.ltype]);
    };
    if (C > 8) {
      std::atomic<int>& big = g_big_cluster[wide][a.ltype][dev];
      int known = big.load(std::memory_order_relaxed);
      if (!known) {
        int n = 0;
        const int keep = C;
        C = kMaxCluster;
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) shape();
        known = e == cudaSuccess && cudaOccupancyMaxActiveClusters(&n, fn, &cfg) == cudaSuccess && n >= 1 ? 2 : 1;
        (void)cudaGetLastError();
        big.store(known, std::memory_order_relaxed);
        C = keep;
      }
      if (known != 2) C = std::max(8, need);
    }
    shape();
    if (e != cudaSuccess) return e;
    return cudaLaunchKernelEx(&cfg, kernel, a, (nvec + C - 1) / C);
  });
}

}  // namespace nls
