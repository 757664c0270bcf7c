// nls_g4.cu -- nls_g4_matmul: y[b][r] = sum_c w(r, c) x[b][c] for 4-bit
// weights with a scale (and minimum) per group of columns, on the 5th-
// generation tensor cores.
//
// With q' = q - 8 and, where there are minimums, m' = m + 8 s:
//   y[b][r] = sum_g ( s[g][r] * sum_{c in g} q'[r][c] x[b][c]
//                     + m'[g][r] * sum_{c in g} x[b][c] )
// q' is exact in fp16 and bfloat16, so tcgen05.mma kind::f16 forms the inner
// sums from exact products with fp32 accumulation, and the scales stay in fp32
// outside them: no weight is rounded. fp32 activations are split into three
// bfloat16 parts that hold all 24 bits, multiplied one after the other into
// the same accumulator. fp32 and bfloat16 activations enter as x 2^-12, and
// the result is multiplied by 2^12: 128 products with q' reach 2^10 times the
// largest activation, which would pass fp32's range before the scales bring it
// down.
//
// What bounds it: at a few batch rows the weights' bytes (half a byte per
// weight); turning them into operands is the work per byte. So the A operand
// never touches shared memory: a thread owns a weight row, reads its packed
// bytes from the staged tile, turns a 32-bit word into four packed pairs
// (4 logical operations, 1-3 shifts and 4 packed fp16/bf16 operations per 8
// weights) and stores them to tensor memory (tcgen05.st), from where the MMA
// reads A; the sums come back to the same thread (tcgen05.ld), whose row's
// scale is then one register. The K order inside a word is the unpacking's
// (0 4 1 5 2 6 3 7); the activations are laid out in that order once per call.
//
// Work: a tile is 256 weight rows (two MMAs of M = 128), a step 128 columns of
// it. The steps of all tiles, in order, are dealt out evenly to the CTAs (one
// per SM), so an SM's load is within one step of every other's whatever the
// shape; a tile that more than one CTA worked on is joined by the last of them
// to finish, from partial sums in the workspace added in CTA order (the same
// bits every time; no CTA waits for another).
// One CTA: 16 worker warps (warp w: lanes 32 (w & 3) .. of tile half (w >> 2)
// & 1, columns of half w >> 3 of the step and of the batch) and one warp that
// issues the copies (a ring of stages: packed weights by tensor map,
// activations, scales) and the MMAs. Workers unpack step s while the MMAs of
// step s - 1 run, then add step s - 1's sums; operands and accumulators are
// double-buffered in TMEM (2 x 128 and 2 x 128 columns).
#include <cuda.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "nls_kernels.h"
#include "nls_tma.cuh"
#include "nls_types.cuh"

namespace nls {

namespace {

constexpr int kTile = 256;       // weight rows per tile
constexpr int kStep = 128;       // columns per step
constexpr int kWorkers = 16;     // warps
constexpr int kThreads = 32 * (kWorkers + 1);
constexpr int kRawBytes = kTile * kStep / 2;
constexpr int kMaxStages = 8;
constexpr int kMaxN = 64;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemD = 256;  // A buffers below, accumulators from here on

// MMA columns of a launch of nb batch rows, and batch rows per worker thread
// (a worker takes one half of them)
__host__ __device__ constexpr int cols_per_thread(int nb) {
  return nb <= 2 ? 1 : nb <= 4 ? 2 : nb <= 8 ? 4 : nb <= 16 ? 8 : nb <= 32 ? 16 : nb <= 48 ? 24 : 32;
}
__host__ __device__ constexpr int mma_n(int cpt) { return cpt <= 8 ? 16 : 2 * cpt; }
// groups (scales) per step, and the most batch rows a launch takes with them:
// each has 64 / regions accumulator columns of the 64 a tile half's buffer holds
__host__ __device__ constexpr int regions_of(int group) { return group == 32 ? 4 : group == 64 ? 2 : 1; }

struct Plan {
  int ksteps, tiles, grid;
  int64_t steps;                 // tiles * ksteps
  int parts;                     // bfloat16 parts of an activation: 3 for fp32
  int regions;
  int nmax;                      // batch rows per launch
  // workspace
  size_t x_bytes, sum_bytes, part_bytes, count_bytes;
  size_t total() const { return x_bytes + sum_bytes + part_bytes + count_bytes; }
};

Plan plan_of(const G4Args& a, int sm_count) {
  Plan p;
  p.ksteps = (a.cols + kStep - 1) / kStep;
  p.tiles = (a.rows + kTile - 1) / kTile;
  p.steps = (int64_t)p.tiles * p.ksteps;
  p.grid = (int)std::min<int64_t>(sm_count, p.steps);
  p.parts = a.xtype == NLS_DT_F32 ? 3 : 1;
  p.regions = regions_of(a.group);
  p.nmax = kMaxN / p.regions;
  const int n = mma_n(cols_per_thread(std::min(a.nb, p.nmax)));
  p.x_bytes = (size_t)p.ksteps * p.parts * n * (kStep * 2);
  p.sum_bytes = a.mins ? (size_t)p.ksteps * p.regions * n * sizeof(float) : 0;
  p.part_bytes = (size_t)p.grid * 2 * n * kTile * sizeof(float);
  p.count_bytes = ((size_t)p.tiles * sizeof(int) + 15) & ~size_t(15);
  return p;
}

struct KernelArgs {
  const void* scales;
  const void* mins;
  int64_t s_ld;
  int rows, cols, group, ngroups, ssize, stype;
  int nb;
  const uint8_t* x;     // laid-out activations, ksteps x parts x N x 256 bytes
  const float* xsum;    // their sums [ksteps][regions][N]
  float* part;          // partial tiles [2 * grid][N][256]
  int* count;           // steps joined so far, per tile
  void* y;
  int ytype;
  int64_t ldy;
  float out_scale;
  int ksteps, parts, stages, stage_bytes, x_off, s_off, m_off;
  int64_t steps;
  unsigned long long wait_ns;
  int* status;
};

// ---- the activations' layout ------------------------------------------------
// One block per step; a thread takes 8 columns of a batch row and writes them,
// permuted, as one 16-byte line of the operand (no-swizzle K-major: 8 rows x 16
// bytes per core matrix, K step j of 16 columns at j * N * 32), for each part.
// With minimums it also sums them per region (the 16 threads of a batch row
// are neighbours). Rows nb .. N - 1 and columns past the matrix are zeros. The
// first block clears the status and the tiles' counters.
template <class X>
__global__ void __launch_bounds__(1024) g4_layout_kernel(const X* x, int64_t ldx, int nb, int n_cols, int cols,
                                                         int parts, int regions, uint8_t* op, float* xsum,
                                                         int* count, int tiles, int* status, int clear_status) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int k = blockIdx.x, n = threadIdx.x >> 4, word = threadIdx.x & 15;
  if (k == 0) {
    if (threadIdx.x == 0 && clear_status) *status = NLS_OK;
  }
  for (int i = k * (int)blockDim.x + (int)threadIdx.x; i < tiles; i += (int)(gridDim.x * blockDim.x)) count[i] = 0;
  constexpr bool kF32 = std::is_same<X, float>::value;
  constexpr float kIn = std::is_same<X, __half>::value ? 1.0f : 0x1p-12f;
  const int c0 = k * kStep + word * 8;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.0f;
  if (n < nb && c0 < cols) {  // (columns come in whole 32)
    const X* p = x + (int64_t)n * ldx + c0;
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      X t[8];
#pragma unroll
      for (int e = 0; e < (int)(8 * sizeof(X) / 16); ++e) reinterpret_cast<uint4*>(t)[e] = reinterpret_cast<const uint4*>(p)[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = to_f32(t[e]) * kIn;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = to_f32(p[e]) * kIn;
    }
  }
  if (xsum) {
    float s = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    const int lanes = 16 / regions;
    for (int o = 1; o < lanes; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (word % lanes == 0) xsum[((size_t)k * regions + word / lanes) * n_cols + n] = s;
  }
  constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};
  uint8_t* dst = op + (size_t)k * parts * n_cols * (kStep * 2) + (size_t)(word >> 1) * (n_cols * 32) +
                 (n >> 3) * 256 + (word & 1) * 128 + (n & 7) * 16;
#pragma unroll
  for (int part = 0; part < (kF32 ? 3 : 1); ++part) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t h[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float& f = v[kOrder[2 * j + e]];
        if constexpr (kF32) {
          // the leading 8 bits, cut off (so that the largest values do not
          // round up to infinity); what is left is exact
          const uint32_t u = __float_as_uint(f);
          const bool fin = (u & 0x7f800000u) != 0x7f800000u;
          h[e] = fin ? u >> 16 : __bfloat16_as_ushort(__float2bfloat16_rn(f));
          f = fin ? f - __uint_as_float(u & 0xffff0000u) : 0.0f;
        } else if constexpr (std::is_same<X, __half>::value) {
          h[e] = __half_as_ushort(__float2half_rn(f));
        } else {
          h[e] = __bfloat16_as_ushort(__float2bfloat16_rn(f));
        }
      }
      w[j] = h[0] | (h[1] << 16);
    }
    *reinterpret_cast<uint4*>(dst + (size_t)part * n_cols * (kStep * 2)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- the product ------------------------------------------------------------

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// D (+)= A . B^T, A in tensor memory, B by descriptor
__device__ __forceinline__ void mma_f16(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t t, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// C consecutive columns of this warp's lanes
template <int C>
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t* r) {
  if constexpr (C == 1) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r[0]) : "r"(t));
  } else if constexpr (C == 2) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(t));
  } else if constexpr (C == 4) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(t));
  } else {
    static_assert(C == 8, "1, 2, 4 or 8 columns");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(t));
  }
}

// the eight weights of a word as q - 8, in pairs (0, 4) (1, 5) (2, 6) (3, 7):
// a nibble under the exponent of 2^10 (fp16) or 2^7 (bfloat16) is that power
// plus q, exactly; fp16's 10 bits of mantissa take the nibble at bit 4 too, as
// 2^10 + 16 q
template <bool BF16>
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t* o) {
  if constexpr (BF16) {
    const __nv_bfloat162 c = __floats2bfloat162_rn(136.0f, 136.0f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t t = ((w >> (4 * j)) & 0x000F000Fu) | 0x43004300u;
      const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&t), c);
      o[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else {
    const __half2 c = __floats2half2_rn(1032.0f, 1032.0f);
    const __half2 k = __floats2half2_rn(0.0625f, 0.0625f), d = __floats2half2_rn(-72.0f, -72.0f);
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const uint32_t v = w >> (4 * j);
      const uint32_t t0 = (v & 0x000F000Fu) | 0x64006400u, t1 = (v & 0x00F000F0u) | 0x64006400u;
      const __half2 h0 = __hsub2(*reinterpret_cast<const __half2*>(&t0), c);
      const __half2 h1 = __hfma2(*reinterpret_cast<const __half2*>(&t1), k, d);
      o[j] = *reinterpret_cast<const uint32_t*>(&h0);
      o[j + 1] = *reinterpret_cast<const uint32_t*>(&h1);
    }
  }
}

__device__ __forceinline__ float ld_scale(const uint8_t* base, int stype, int i) {
  if (stype == NLS_DT_F32) return reinterpret_cast<const float*>(base)[i];
  if (stype == NLS_DT_F16) return __half2float(reinterpret_cast<const __half*>(base)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
}

__device__ __forceinline__ void st_out(void* y, int ytype, int64_t i, float v) {
  if (ytype == NLS_DT_F32) reinterpret_cast<float*>(y)[i] = v;
  else if (ytype == NLS_DT_F16) reinterpret_cast<__half*>(y)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
}

struct Bars {
  uint64_t full[kMaxStages];  // stage landed
  uint64_t ready[2];          // every worker has stored step s's operand (s & 1)
  uint64_t done[2];           // step s's MMAs have completed
  uint64_t joined;            // every worker has written its partial sums
  uint64_t told;              // whether this CTA is the tile's last
  uint32_t tmem;
  int fail, staged, issued, last;
};

template <bool BF16, int CPT, int R>
__global__ void __launch_bounds__(kThreads, 1)
    g4_kernel(const KernelArgs a, const __grid_constant__ CUtensorMap qmap) {
  constexpr int N = mma_n(CPT);
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars& B = *reinterpret_cast<Bars*>(smem + (size_t)a.stages * a.stage_bytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t s0 = a.steps * blockIdx.x / gridDim.x, s1 = a.steps * (blockIdx.x + 1) / gridDim.x;
  const int nsteps = (int)(s1 - s0);
  const int tile0 = (int)(s0 / a.ksteps), k0 = (int)(s0 % a.ksteps);

  if (tid == 0) {
    for (int i = 0; i < kMaxStages; ++i) mbar_init(&B.full[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B.ready[i], kWorkers);
      mbar_init(&B.done[i], 1);
    }
    mbar_init(&B.joined, kWorkers);
    mbar_init(&B.told, 1);
    B.fail = 0;
    B.staged = B.issued = -1;
    fence_mbar_init();
  }
  if (warp == kWorkers) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tbase = B.tmem;
  // the laid-out activations, their sums and the cleared counters are there
  asm volatile("griddepcontrol.wait;" ::: "memory");

  bool fail = false;
  if (warp == kWorkers) {
    if (lane == 0) {
      int ltile = tile0, lk = k0;  // position of the next step to stage
      auto stage = [&](int s) {
        if (s >= nsteps) return;
        uint8_t* st = smem + (size_t)(s % a.stages) * a.stage_bytes;
        uint64_t* bar = &B.full[s % a.stages];
        const int r0 = ltile * kTile, g0 = (int)((int64_t)lk * kStep / a.group);
        const uint32_t xb = (uint32_t)(a.parts * N * kStep * 2);
        const uint32_t line = (uint32_t)(min(kTile, (a.rows - r0 + 7) & ~7) * a.ssize);
        const int ng = min(R, a.ngroups - g0);
        mbar_arrive_expect_tx(bar, kRawBytes + xb + (uint32_t)ng * line * (a.mins ? 2u : 1u));
        tma_load_2d(st, &qmap, lk * (kStep / 2), r0, bar);
        bulk_copy_g2s(st + a.x_off, a.x + (size_t)lk * xb, xb, bar);
        for (int g = 0; g < ng; ++g) {
          const size_t at = ((size_t)(g0 + g) * a.s_ld + r0) * a.ssize;
          bulk_copy_g2s(st + a.s_off + g * kTile * a.ssize, static_cast<const uint8_t*>(a.scales) + at, line, bar);
          if (a.mins)
            bulk_copy_g2s(st + a.m_off + g * kTile * a.ssize, static_cast<const uint8_t*>(a.mins) + at, line, bar);
        }
        B.staged = s;
        if (++lk == a.ksteps) {
          lk = 0;
          ++ltile;
        }
      };
      const uint32_t idesc = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) |
                             ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      for (int s = 0; s < a.stages; ++s) stage(s);
      for (int s = 0; s < nsteps; ++s) {
        if (!mbar_wait_bounded(&B.ready[s & 1], (uint32_t)((s >> 1) & 1), a.wait_ns)) {
          fail = true;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t xs = smem_u32(smem) + (uint32_t)((s % a.stages) * a.stage_bytes + a.x_off);
        // no-swizzle K-major descriptor: 128 bytes from a row's first 8
        // columns to its next 8, 256 from 8 rows to the next
        const uint64_t bd = (uint64_t)((xs >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 16) |
                            ((uint64_t)(256 >> 4) << 32) | ((uint64_t)1 << 46);
        for (int t = 0; t < 2; ++t) {
          const uint32_t ta = tbase + (uint32_t)(((s & 1) * 2 + t) * 64);
          const uint32_t td = tbase + kTmemD + (uint32_t)(((s & 1) * 2 + t) * 64);
          for (int p = 0; p < a.parts; ++p) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              mma_f16(td + (uint32_t)(j * R / 8 * N), ta + 8 * j, bd + (uint64_t)((p * 8 + j) * (N * 32) / 16), idesc,
                      (p > 0 || j % (8 / R) != 0) ? 1u : 0u);
          }
        }
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                         smem_u32(&B.done[s & 1]))
                     : "memory");
        B.issued = s;
        // step s - 1's stage is free once its MMAs have read its activations
        // (its weights and scales were read before they were issued)
        if (s > 0 && s - 1 + a.stages < nsteps) {
          if (!mbar_wait_bounded(&B.done[(s - 1) & 1], (uint32_t)(((s - 1) >> 1) & 1), a.wait_ns)) {
            fail = true;
            break;
          }
          stage(s - 1 + a.stages);
        }
      }
    }
    fail = __any_sync(0xffffffffu, fail);
  } else {
    const int quarter = warp & 3, t = (warp >> 2) & 1, half = warp >> 3;
    const int row = t * 128 + quarter * 32 + lane;  // in the tile
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    float acc[CPT], sc[R], mn[R], nsc[R], nmn[R];
#pragma unroll
    for (int j = 0; j < CPT; ++j) acc[j] = 0.0f;
    int ends = 0;  // tiles joined so far (phase of the joining barriers)
    int tile = tile0, k = k0;  // position of the step being added
    int uk = k0;               // column step being unpacked

    // adds step s's sums; at the end of a tile, or of this CTA's steps, writes
    auto add = [&](int s) -> bool {
      if (__any_sync(0xffffffffu, !mbar_wait_bounded(&B.done[s & 1], (uint32_t)((s >> 1) & 1), a.wait_ns))) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t td = tbase + kTmemD + lanes + (uint32_t)(((s & 1) * 2 + t) * 64 + half * CPT);
      constexpr int C = CPT < 8 ? CPT : 8;
#pragma unroll
      for (int c = 0; c < CPT; c += C) {
        uint32_t d[R][C];
#pragma unroll
        for (int r = 0; r < R; ++r) tmem_ld<C>(td + (uint32_t)(r * N + c), d[r]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < C; ++j) acc[c + j] = __fmaf_rn(sc[r], __uint_as_float(d[r][j]), acc[c + j]);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      if (a.mins) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float* xs = a.xsum + ((size_t)k * R + r) * N + half * CPT;
#pragma unroll
          for (int j = 0; j < CPT; ++j) acc[j] = __fmaf_rn(mn[r], xs[j], acc[j]);
        }
      }
      if (k + 1 < a.ksteps && s + 1 < nsteps) {
        ++k;
        return true;
      }
      // the tile's steps of this CTA were [first, k]
      const int first = tile == tile0 ? k0 : 0;
      const int r = tile * kTile + row;
      bool write = true;
      if (first != 0 || k + 1 != a.ksteps) {
        float* mine = a.part + ((size_t)(2 * blockIdx.x + (tile == tile0 ? 0 : 1)) * N + half * CPT) * kTile + row;
#pragma unroll
        for (int j = 0; j < CPT; ++j) __stcg(mine + j * kTile, acc[j]);
        __threadfence();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.joined);
        const uint32_t ph = (uint32_t)(ends & 1);
        if (warp == 0) {
          if (__any_sync(0xffffffffu, !mbar_wait_bounded(&B.joined, ph, a.wait_ns))) return false;
          if (lane == 0) {
            __threadfence();
            const int had = atomicAdd(a.count + tile, k + 1 - first);
            __threadfence();
            B.last = had + (k + 1 - first) == a.ksteps;
            mbar_arrive(&B.told);
          }
        }
        if (__any_sync(0xffffffffu, !mbar_wait_bounded(&B.told, ph, a.wait_ns))) return false;
        ++ends;
        write = B.last != 0;
        if (write) {
          // every contributor's sums, in the order of the CTAs: the first is
          // the one whose steps hold the tile's first step
          const int64_t lo = (int64_t)tile * a.ksteps;
          int c = (int)(((lo + 1) * gridDim.x - 1) / a.steps);
#pragma unroll
          for (int j = 0; j < CPT; ++j) acc[j] = 0.0f;
          for (;; ++c) {
            const int64_t b0 = a.steps * c / gridDim.x;
            if (b0 >= lo + a.ksteps) break;
            const float* theirs = a.part + ((size_t)(2 * c + (b0 >= lo ? 0 : 1)) * N + half * CPT) * kTile + row;
#pragma unroll
            for (int j = 0; j < CPT; ++j) acc[j] = __fadd_rn(acc[j], __ldcg(theirs + j * kTile));
            if (c + 1 == (int)gridDim.x) break;
          }
        }
      }
      if (write && r < a.rows) {
#pragma unroll
        for (int j = 0; j < CPT; ++j)
          if (half * CPT + j < a.nb) st_out(a.y, a.ytype, (int64_t)(half * CPT + j) * a.ldy + r, acc[j] * a.out_scale);
      }
#pragma unroll
      for (int j = 0; j < CPT; ++j) acc[j] = 0.0f;
      ++tile;
      k = 0;
      return true;
    };

    for (int s = 0; s < nsteps; ++s) {
      const uint8_t* st = smem + (size_t)(s % a.stages) * a.stage_bytes;
      if (__any_sync(0xffffffffu, !mbar_wait_bounded(&B.full[s % a.stages], (uint32_t)((s / a.stages) & 1), a.wait_ns))) {
        fail = true;
        break;
      }
      uint32_t raw[8];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        // 16-byte pieces of a 64-byte row lie where the 64-byte swizzle of
        // the copy put them (free of bank conflicts)
        const uint4 v = *reinterpret_cast<const uint4*>(st + row * 64 + (((2 * half + c) ^ ((row >> 1) & 3)) << 4));
        raw[4 * c] = v.x;
        raw[4 * c + 1] = v.y;
        raw[4 * c + 2] = v.z;
        raw[4 * c + 3] = v.w;
      }
      const int g0 = (int)((int64_t)uk * kStep / a.group);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool in = g0 + r < a.ngroups;  // (a short last step has fewer groups)
        nsc[r] = in ? ld_scale(st + a.s_off, a.stype, r * kTile + row) : 0.0f;
        nmn[r] = in && a.mins ? __fmaf_rn(8.0f, nsc[r], ld_scale(st + a.m_off, a.stype, r * kTile + row)) : 0.0f;
      }
      if (++uk == a.ksteps) uk = 0;
      uint32_t o[32];
#pragma unroll
      for (int i = 0; i < 8; ++i) unpack8<BF16>(raw[i], o + 4 * i);
      tmem_st32(tbase + lanes + (uint32_t)(((s & 1) * 2 + t) * 64 + half * 32), o);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.ready[s & 1]);
      if (s > 0 && !add(s - 1)) {
        fail = true;
        break;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        sc[r] = nsc[r];
        mn[r] = nmn[r];
      }
    }
    if (!fail && nsteps > 0 && !add(nsteps - 1)) fail = true;
  }
  if (fail) B.fail = 1;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (B.fail) {
    if (tid == 0) {
      atomicCAS(a.status, 0, NLS_ERR_TIMEOUT);
      // copies and MMAs in flight finish before their memory is released
      // (under the default limit: they are real)
      for (int s = max(0, B.staged - a.stages + 1); s <= B.staged; ++s)
        (void)mbar_wait_bounded(&B.full[s % a.stages], (uint32_t)((s / a.stages) & 1));
      for (int s = max(0, B.issued - 1); s <= B.issued; ++s)
        (void)mbar_wait_bounded(&B.done[s & 1], (uint32_t)((s >> 1) & 1));
    }
    __syncthreads();
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == kWorkers)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(kTmemCols) : "memory");
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (EncodeTiledFn) nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}


template <bool BF16, int R>
const void* kernel_of(int cpt) {
  switch (cpt) {
    case 1: return (const void*)g4_kernel<BF16, 1, R>;
    case 2: return (const void*)g4_kernel<BF16, 2, R>;
    case 4: return (const void*)g4_kernel<BF16, 4, R>;
    case 8: return (const void*)g4_kernel<BF16, 8, R>;
  }
  if constexpr (R <= 2) {
    if (cpt == 16) return (const void*)g4_kernel<BF16, 16, R>;
  }
  if constexpr (R == 1) {
    if (cpt == 24) return (const void*)g4_kernel<BF16, 24, R>;
    if (cpt == 32) return (const void*)g4_kernel<BF16, 32, R>;
  }
  return nullptr;
}

}  // namespace

size_t g4_workspace_bytes(const G4Args& a, int sm_count) { return plan_of(a, sm_count).total(); }

cudaError_t launch_g4(const G4Args& a, void* workspace, int sm_count, cudaStream_t st) {
  const Plan p = plan_of(a, sm_count);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  CUtensorMap map;
  memset(&map, 0, sizeof map);
  const EncodeTiledFn enc = encode_tiled();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)(a.cols / 2), (cuuint64_t)a.rows};
  const cuuint64_t strides[1] = {(cuuint64_t)a.q_ld};
  const cuuint32_t box[2] = {kStep / 2, kTile};
  const cuuint32_t ones[2] = {1, 1};
  if (enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(a.q), dims, strides, box, ones,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;

  KernelArgs k{};
  k.scales = a.scales;
  k.mins = a.mins;
  k.s_ld = a.s_ld;
  k.rows = a.rows;
  k.cols = a.cols;
  k.group = a.group;
  k.ngroups = (a.cols + a.group - 1) / a.group;
  k.stype = a.stype;
  k.ssize = (int)dt_size(a.stype);
  k.x = ws;
  k.xsum = a.mins ? reinterpret_cast<float*>(ws + p.x_bytes) : nullptr;
  k.part = reinterpret_cast<float*>(ws + p.x_bytes + p.sum_bytes);
  k.count = reinterpret_cast<int*>(ws + p.x_bytes + p.sum_bytes + p.part_bytes);
  k.ytype = a.ytype;
  k.ldy = a.ldy;
  k.out_scale = a.xtype == NLS_DT_F16 ? 1.0f : 4096.0f;
  k.ksteps = p.ksteps;
  k.parts = p.parts;
  k.steps = p.steps;
  k.wait_ns = a.wait_ns;
  k.status = a.status;
  const bool bf16 = a.xtype != NLS_DT_F16;
  const size_t xes = dt_size(a.xtype), yes = dt_size(a.ytype);
  for (int b0 = 0; b0 < a.nb; b0 += p.nmax) {
    k.nb = std::min(p.nmax, a.nb - b0);
    const int cpt = cols_per_thread(k.nb), n = mma_n(cpt);
    k.y = static_cast<uint8_t*>(a.y) + (size_t)b0 * a.ldy * yes;
    k.x_off = kRawBytes;
    k.s_off = k.x_off + p.parts * n * kStep * 2;
    k.m_off = k.s_off + p.regions * kTile * k.ssize;
    k.stage_bytes = (k.m_off + (a.mins ? p.regions * kTile * k.ssize : 0) + 1023) & ~1023;
    const int room = 227 * 1024 - 1024 - (int)sizeof(Bars);
    k.stages = std::min(kMaxStages, room / k.stage_bytes);
    const size_t smem = (size_t)k.stages * k.stage_bytes + sizeof(Bars);
    const void* kern = p.regions == 4 ? (bf16 ? kernel_of<true, 4>(cpt) : kernel_of<false, 4>(cpt))
                       : p.regions == 2 ? (bf16 ? kernel_of<true, 2>(cpt) : kernel_of<false, 2>(cpt))
                                        : (bf16 ? kernel_of<true, 1>(cpt) : kernel_of<false, 1>(cpt));
    if (!kern) return cudaErrorInvalidValue;
    const void* x = static_cast<const uint8_t*>(a.x) + (size_t)b0 * a.ldx * xes;
    with_type(a.xtype, [&](auto xv) {
      using X = decltype(xv);
      g4_layout_kernel<X><<<p.ksteps, 16 * n, 0, st>>>(static_cast<const X*>(x), a.ldx, k.nb, n, a.cols, p.parts,
                                                       p.regions, ws, const_cast<float*>(k.xsum), k.count, p.tiles,
                                                       a.status, b0 == 0);
    });
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void* args[2] = {&k, &map};
    e = cudaLaunchKernelExC(&cfg, kern, args);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace nls
