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
// Work: a tile is 256 weight rows (two MMAs of M = 128), a step 256 columns of
// it: 128 bytes of a row, since the copy of a step costs the copy engine about
// 4 cycles a row however short the row (64-byte rows held the kernel to 3.4
// TB/s). The steps of all tiles, in order, are dealt out evenly to the CTAs (one
// per SM), so an SM's load is within one step of every other's whatever the
// shape; a tile that more than one CTA worked on is joined by the last of them
// to finish, from partial sums in the workspace added in CTA order (the same
// bits every time; no CTA waits for another).
// One CTA, 26 warps: 16 unpack in two sets, each one half of a step's columns (a
// thread 128 columns of its row); 8 add the halves' sums to their rows'; one
// issues the copies (a ring of stages: packed weights by tensor map,
// activations, scales) and one the MMAs. Roles only wait for one another
// through mbarriers, and each runs as far ahead as its buffers let it: operands
// have one buffer per set in TMEM (2 x 128 columns), accumulators as many as
// fit in the other 256 columns.
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
constexpr int kHalf = 128;       // columns per half of a step
constexpr int kStep = 2 * kHalf;  // columns per step
constexpr int kUnpackWarps = 16;  // two sets
constexpr int kAddWarps = 8;
constexpr int kCopyWarp = kUnpackWarps + kAddWarps, kMmaWarp = kCopyWarp + 1;
constexpr int kThreads = 32 * (kMmaWarp + 1);
constexpr int kRawBytes = kTile * kStep / 2;
constexpr int kMaxStages = 8;
constexpr int kMaxN = 64;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemD = 256;  // A buffers below, accumulators from here on

// batch rows a launch is compiled for, and the MMA's columns. fp32 activations'
// three parts are columns of their own up to 4 batch rows.
__host__ __device__ constexpr int batch_of(int nb) {
  return nb <= 1 ? 1 : nb <= 2 ? 2 : nb <= 4 ? 4 : nb <= 8 ? 8 : nb <= 16 ? 16 : nb <= 32 ? 32 : nb <= 48 ? 48 : 64;
}
__host__ __device__ constexpr int mma_n(int nbt) { return nbt <= 16 ? 16 : nbt; }
__host__ __device__ constexpr bool folded(int parts, int nb) { return parts == 3 && nb <= 4; }
// groups (scales) per half step; its accumulators take regions x N columns per
// tile half, 64 at most
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
  // (fp32's three parts: a stage of 64 rows would leave room for one stage only)
  p.nmax = std::min(kMaxN / p.regions, p.parts == 3 ? 32 : kMaxN);
  const int n = mma_n(batch_of(std::min(a.nb, p.nmax)));
  p.x_bytes = (size_t)p.ksteps * p.parts * n * (kStep * 2);
  p.sum_bytes = a.mins ? (size_t)p.ksteps * 2 * p.regions * n * sizeof(float) : 0;
  p.part_bytes = (size_t)p.grid * 2 * n * kTile * sizeof(float);
  p.count_bytes = ((size_t)p.tiles * sizeof(int) + 15) & ~size_t(15);
  return p;
}

struct KernelArgs {
  const void* scales;
  const void* mins;
  int64_t s_ld;
  int rows, group, ssize, stype;
  int lines;            // lines of scales as the halves use them: of whole groups up to 128 wide, else per half
  int nb;
  const uint8_t* x;     // laid-out activations, per half step parts x N x 256 bytes
  const float* xsum;    // their sums [half step][regions][N]
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
// One block per half step; a thread takes 8 columns of a batch row and writes them,
// permuted, as one 16-byte line of the operand (no-swizzle K-major: 8 rows x 16
// bytes per core matrix, K step j of 16 columns at j * N * 32), for each part.
// With minimums it also sums them per region (the 16 threads of a batch row
// are neighbours). Rows nb .. N - 1 and columns past the matrix are zeros. The
// first block clears the status and the tiles' counters.
template <class X>
__global__ void __launch_bounds__(1024) g4_layout_kernel(const X* x, int64_t ldx, int nb, int n_cols, int cols,
                                                         int parts, int fold, int regions, uint8_t* op, float* xsum,
                                                         int* count, int tiles, int* status, int clear_status) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int k = blockIdx.x, n = threadIdx.x >> 4, word = threadIdx.x & 15;
  if (k == 0) {
    if (threadIdx.x == 0 && clear_status) *status = NLS_OK;
  }
  for (int i = k * (int)blockDim.x + (int)threadIdx.x; i < tiles; i += (int)(gridDim.x * blockDim.x)) count[i] = 0;
  constexpr bool kF32 = std::is_same<X, float>::value;
  constexpr float kIn = std::is_same<X, __half>::value ? 1.0f : 0x1p-12f;
  const int c0 = k * kHalf + word * 8;
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
  // fold > 0: part p of batch row n is column p * fold + n (columns past the
  // parts are zeros: threads n >= fold write them)
  uint8_t* dst = op + (size_t)k * (fold ? 1 : parts) * n_cols * (kHalf * 2) + (size_t)(word >> 1) * (n_cols * 32) +
                 (word & 1) * 128;
  auto line = [&](int c) { return dst + (c >> 3) * 256 + (c & 7) * 16; };
  if (fold && n >= fold) {
    if (n >= 3 * fold) *reinterpret_cast<uint4*>(line(n)) = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
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
    uint8_t* at = fold ? line(part * fold + n) : line(n) + (size_t)part * n_cols * (kHalf * 2);
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
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

// D (+)= A . B^T by the warp's leader, A in tensor memory, B by descriptor. The
// whole warp gets here with the same values: behind a branch of one lane the
// operands would have to be moved to uniform registers one by one, which made
// an issue cost about 110 cycles.
template <bool ACC>
__device__ __forceinline__ void mma_f16(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %4, 0;\n\t"
      "setp.ne.u32 p, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(leader), "n"(ACC ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
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
struct Unpack {
  // the power of two's bits, out of the compiler's sight: as an immediate it
  // would take a logical operation of its own beside the mask's
  uint32_t magic;
  __device__ __forceinline__ Unpack() { asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(BF16 ? 0x43004300 : 0x64006400)); }
  template <uint32_t MASK>
  __device__ __forceinline__ uint32_t put(uint32_t w) const {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(MASK), "r"(magic));  // (w & MASK) | magic
    return r;
  }
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t* o) const {
    if constexpr (BF16) {
      const __nv_bfloat162 c = __floats2bfloat162_rn(136.0f, 136.0f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t t = put<0x000F000Fu>(w >> (4 * j));
        const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&t), c);
        o[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    } else {
      const __half2 c = __floats2half2_rn(1032.0f, 1032.0f);
      const __half2 k = __floats2half2_rn(0.0625f, 0.0625f), d = __floats2half2_rn(-72.0f, -72.0f);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const uint32_t v = w >> (4 * j);
        const uint32_t t0 = put<0x000F000Fu>(v), t1 = put<0x00F000F0u>(v);
        const __half2 h0 = __hsub2(*reinterpret_cast<const __half2*>(&t0), c);
        const __half2 h1 = __hfma2(*reinterpret_cast<const __half2*>(&t1), k, d);
        o[j] = *reinterpret_cast<const uint32_t*>(&h0);
        o[j + 1] = *reinterpret_cast<const uint32_t*>(&h1);
      }
    }
  }
};

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

constexpr int kMaxBuffers = 8;  // accumulator buffers

struct Bars {
  uint64_t full[kMaxStages];    // stage landed
  uint64_t free[kMaxStages];    // the step's sums are added (its MMAs are done, its scales read)
  uint64_t ready[2];            // the set has stored its half's operand
  uint64_t done[kMaxBuffers];   // a half's MMAs have completed
  uint64_t added[kMaxBuffers];  // its sums have been read
  uint64_t joined;              // every adding warp has written its partial sums
  uint64_t told;                // whether this CTA is the tile's last
  uint32_t tmem;
  int fail, staged, issued, last;
};

// barriers by their shared-memory address (32-bit arithmetic)
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __noinline__ bool warp_wait_slow(uint32_t bar, uint32_t parity, unsigned long long limit_ns) {
  const unsigned long long t0 = globaltimer_ns();
  while (true) {
    if (__all_sync(0xffffffffu, try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, globaltimer_ns() - t0 > limit_ns)) return false;
  }
}
// a whole warp's bounded wait (the same answer in every lane)
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, unsigned long long limit_ns) {
  if (__all_sync(0xffffffffu, try_wait(bar, parity))) return true;
  return warp_wait_slow(bar, parity, limit_ns);
}

// a position in a ring of n and the phase of its barriers there
struct Ring {
  int i;
  uint32_t phase;
  __device__ __forceinline__ void next(int n, int by = 1) {
    i += by;
    if (i >= n) {
      i -= n;
      phase ^= 1;
    }
  }
};

// NB: batch rows. R: groups per step. FOLD: the three parts of fp32 activations
// are columns of their own (part p of batch row b in column NB p + b), else
// further MMAs into the same columns.
template <bool BF16, int NB, int R, bool FOLD>
__global__ void __launch_bounds__(kThreads, 1)
    g4_kernel(const KernelArgs a, const __grid_constant__ CUtensorMap qmap) {
  constexpr int N = mma_n(NB);
  constexpr int P = FOLD ? 3 : 1;
  constexpr int kBuffers = 128 / (R * N) < kMaxBuffers ? 128 / (R * N) : kMaxBuffers;
  static_assert(NB * P <= N && R * N <= 64 && kBuffers >= 2, "columns");
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars& B = *reinterpret_cast<Bars*>(smem + (size_t)a.stages * a.stage_bytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t s0 = a.steps * blockIdx.x / gridDim.x, s1 = a.steps * (blockIdx.x + 1) / gridDim.x;
  const int nsteps = (int)(s1 - s0);
  const int tile0 = (int)(s0 / a.ksteps), k0 = (int)(s0 % a.ksteps);
  const uint32_t sbase = smem_u32(smem);
  const uint32_t full0 = smem_u32(B.full), free0 = smem_u32(B.free), ready0 = smem_u32(B.ready), done0 = smem_u32(B.done),
                 added0 = smem_u32(B.added);

  if (tid == 0) {
    for (int i = 0; i < kMaxStages; ++i) {
      mbar_init(&B.full[i], 1);
      mbar_init(&B.free[i], kAddWarps);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&B.ready[i], kUnpackWarps / 2);
    for (int i = 0; i < kMaxBuffers; ++i) {
      mbar_init(&B.done[i], 1);
      mbar_init(&B.added[i], kAddWarps);
    }
    mbar_init(&B.joined, kAddWarps);
    mbar_init(&B.told, 1);
    B.fail = 0;
    B.staged = B.issued = -1;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
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

  // (a limit of 0 is a deadline already past: every role but the copies, whose
  // first steps wait for nothing, gives up before its first wait)
  bool fail = a.wait_ns == 0 && warp != kCopyWarp;
  if (fail) {
  } else if (warp == kCopyWarp) {
    if (lane == 0) {
      // position of the next step; its stage and the phase its last step left
      // there; where groups are at least as wide as a half, the next half's
      // group and the halves left in it
      int ltile = tile0, lk = k0;
      Ring slot{0, 1};
      const int per = R == 1 ? a.group / kHalf : 1;
      int g1 = 2 * k0 / per, left = per - 2 * k0 % per;
      const uint32_t xb = (uint32_t)(a.parts * N * kStep * 2);
      for (int s = 0; s < nsteps; ++s) {
        if (s >= a.stages && !mbar_wait_bounded(&B.free[slot.i], slot.phase, a.wait_ns)) {
          fail = true;
          break;
        }
        uint8_t* st = smem + (size_t)slot.i * a.stage_bytes;
        uint64_t* bar = &B.full[slot.i];
        const int r0 = ltile * kTile;
        const uint32_t line = (uint32_t)(min(kTile, (a.rows - r0 + 7) & ~7) * a.ssize);
        const int n = min(2 * R, a.lines - 2 * R * lk);
        mbar_arrive_expect_tx(bar, kRawBytes + xb + (uint32_t)n * line * (a.mins ? 2u : 1u));
        tma_load_2d(st, &qmap, lk * (kStep / 2), r0, bar);
        bulk_copy_g2s(st + a.x_off, a.x + (size_t)lk * xb, xb, bar);
        for (int i = 0; i < n; ++i) {
          int g = 2 * R * lk + i;
          if (R == 1) {
            g = g1;
            if (--left == 0) {
              left = per;
              ++g1;
            }
          }
          const size_t at = ((size_t)g * a.s_ld + r0) * a.ssize;
          bulk_copy_g2s(st + a.s_off + i * kTile * a.ssize, static_cast<const uint8_t*>(a.scales) + at, line, bar);
          if (a.mins)
            bulk_copy_g2s(st + a.m_off + i * kTile * a.ssize, static_cast<const uint8_t*>(a.mins) + at, line, bar);
        }
        B.staged = s;
        slot.next(a.stages);
        if (++lk == a.ksteps) {
          lk = 0;
          ++ltile;
          g1 = 0;
          left = per;
        }
      }
    }
    fail = __any_sync(0xffffffffu, fail);
  } else if (warp == kMmaWarp) {
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) |
                               ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    // no-swizzle K-major descriptor: 128 bytes from a row's first 8 columns to
    // its next 8, 256 from 8 rows to the next
    const uint64_t bd0 = (uint64_t)(((sbase + (uint32_t)a.x_off) >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 16) |
                         ((uint64_t)(256 >> 4) << 32) | ((uint64_t)1 << 46);
    Ring slot{0, 0}, buf{0, 1};  // stage; accumulators, with the phase of their last use
    for (int s = 0; s < nsteps && !fail; ++s) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!warp_wait(ready0 + (uint32_t)h * 8, (uint32_t)(s & 1), a.wait_ns) ||
            (2 * s + h >= kBuffers && !warp_wait(added0 + (uint32_t)buf.i * 8, buf.phase, a.wait_ns))) {
          fail = true;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t bd = bd0 + (uint64_t)(slot.i * (a.stage_bytes >> 4) + h * a.parts * (N * kHalf * 2 / 16));
        const uint32_t ab = tbase + (uint32_t)(h * 128), db = tbase + kTmemD + (uint32_t)(buf.i * (2 * R * N));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j % (8 / R) == 0)
              mma_f16<false>(db + (t * R + j * R / 8) * N, ab + t * 64 + 8 * j, bd + j * (N * 2), idesc, leader);
            else
              mma_f16<true>(db + (t * R + j * R / 8) * N, ab + t * 64 + 8 * j, bd + j * (N * 2), idesc, leader);
          }
        }
        for (int p = 1; p < a.parts; ++p) {
          const uint64_t bp = bd + (uint64_t)(p * 8 * N * 2);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              mma_f16<true>(db + (t * R + j * R / 8) * N, ab + t * 64 + 8 * j, bp + j * (N * 2), idesc, leader);
        }
        if (leader) {
          asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                           done0 + (uint32_t)buf.i * 8)
                       : "memory");
          B.issued = 2 * s + h;
        }
        __syncwarp();
        buf.next(kBuffers);
      }
      slot.next(a.stages);
    }
  } else if (warp < kUnpackWarps) {
    const int quarter = warp & 3, t = (warp >> 2) & 1, set = warp >> 3;
    const int row = t * 128 + quarter * 32 + lane;  // in the tile
    const uint32_t ta = tbase + ((uint32_t)(32 * quarter) << 16) + (uint32_t)(set * 128 + t * 64);
    const uint32_t bar = ready0 + (uint32_t)set * 8;
    // 16-byte pieces of a 128-byte row lie where the 128-byte swizzle of the
    // copy put them (free of bank conflicts)
    uint32_t at[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) at[c] = sbase + (uint32_t)(row * 128 + (((4 * set + c) ^ (row & 7)) << 4));
    const Unpack<BF16> unpack;
    Ring slot{0, 0}, prev{set, 0};  // stage; accumulators of the step before's half
    for (int s = 0; s < nsteps; ++s) {
      if (!warp_wait(full0 + (uint32_t)slot.i * 8, slot.phase, a.wait_ns)) {
        fail = true;
        break;
      }
      const uint32_t st = (uint32_t)(slot.i * a.stage_bytes);
      slot.next(a.stages);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t o[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t v[4];
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                       : "r"(at[2 * h + c] + st)
                       : "memory");
#pragma unroll
          for (int i = 0; i < 4; ++i) unpack(v[i], o + 16 * c + 4 * i);
        }
        // the step before had the same operand buffer
        if (h == 0 && s >= 1) {
          if (!warp_wait(done0 + (uint32_t)prev.i * 8, prev.phase, a.wait_ns)) {
            fail = true;
            break;
          }
          prev.next(kBuffers, 2);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        tmem_st32(ta + h * 32, o);
      }
      if (fail) break;
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(bar);
    }
  } else {
    const int aw = warp - kUnpackWarps, quarter = aw & 3, t = aw >> 2;
    const int row = t * 128 + quarter * 32 + lane;  // in the tile
    const uint32_t td = tbase + ((uint32_t)(32 * quarter) << 16) + kTmemD + (uint32_t)(t * R * N);
    float acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j] = 0.0f;
    int ends = 0;              // tiles joined so far (phase of the joining barriers)
    int tile = tile0, k = k0;  // position of the step
    Ring slot{0, 0}, buf{0, 0};
    for (int s = 0; s < nsteps; ++s) {
      const uint8_t* st = smem + (uint32_t)(slot.i * a.stage_bytes);
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        // (the stage has landed long since: that wait orders the scales' copies)
        if (!warp_wait(done0 + (uint32_t)buf.i * 8, buf.phase, a.wait_ns) ||
            (h == 0 && !warp_wait(full0 + (uint32_t)slot.i * 8, slot.phase, a.wait_ns))) {
          fail = true;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d0 = td + (uint32_t)(buf.i * (2 * R * N));
        const int l0 = (2 * k + h) * R;  // the half's first line of scales
        constexpr int C = NB < 8 ? NB : 8;
        float sc[R];
#pragma unroll
        for (int c = 0; c < NB; c += C) {
          uint32_t d[R][P][C];
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int p = 0; p < P; ++p) tmem_ld<C>(d0 + (uint32_t)(r * N + p * NB + c), d[r][p]);
          if (c == 0) {
#pragma unroll
            for (int r = 0; r < R; ++r)  // (the last step may have fewer)
              sc[r] = l0 + r < a.lines ? ld_scale(st + a.s_off, a.stype, (h * R + r) * kTile + row) : 0.0f;
          }
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < C; ++j) {
              float v = __uint_as_float(d[r][0][j]);
              if constexpr (FOLD) v = (__uint_as_float(d[r][2][j]) + __uint_as_float(d[r][1][j])) + v;
              acc[c + j] = __fmaf_rn(sc[r], v, acc[c + j]);
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        if (a.mins) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (l0 + r >= a.lines) break;
            const float m = __fmaf_rn(8.0f, sc[r], ld_scale(st + a.m_off, a.stype, (h * R + r) * kTile + row));
            const float* xs = a.xsum + (size_t)(l0 + r) * N;
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[j] = __fmaf_rn(m, xs[j], acc[j]);
          }
        }
        __syncwarp();
        if (lane == 0) {
          arrive(added0 + (uint32_t)buf.i * 8);
          if (h == 1) arrive(free0 + (uint32_t)slot.i * 8);
        }
        buf.next(kBuffers);
      }
      if (fail) break;
      slot.next(a.stages);
      if (k + 1 < a.ksteps && s + 1 < nsteps) {
        ++k;
        continue;
      }
      // the end of a tile, or of this CTA's steps; the tile's steps of this
      // CTA were [first, k]
      const int first = tile == tile0 ? k0 : 0;
      const int r = tile * kTile + row;
      bool write = true;
      if (first != 0 || k + 1 != a.ksteps) {
        float* mine = a.part + (size_t)(2 * blockIdx.x + (tile == tile0 ? 0 : 1)) * N * kTile + row;
#pragma unroll
        for (int j = 0; j < NB; ++j) __stcg(mine + j * kTile, acc[j]);
        __threadfence();
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&B.joined));
        const uint32_t ph = (uint32_t)(ends & 1);
        if (aw == 0) {
          if (!warp_wait(smem_u32(&B.joined), ph, a.wait_ns)) {
            fail = true;
            break;
          }
          if (lane == 0) {
            __threadfence();
            const int had = atomicAdd(a.count + tile, k + 1 - first);
            __threadfence();
            B.last = had + (k + 1 - first) == a.ksteps;
            arrive(smem_u32(&B.told));
          }
          __syncwarp();
        }
        if (!warp_wait(smem_u32(&B.told), ph, a.wait_ns)) {
          fail = true;
          break;
        }
        ++ends;
        write = B.last != 0;
        if (write) {
          // every contributor's sums, in the order of the CTAs: the first is
          // the one whose steps hold the tile's first step
          const int64_t lo = (int64_t)tile * a.ksteps;
          int c = (int)(((lo + 1) * gridDim.x - 1) / a.steps);
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[j] = 0.0f;
          for (;; ++c) {
            const int64_t b0 = a.steps * c / gridDim.x;
            if (b0 >= lo + a.ksteps) break;
            const float* theirs = a.part + (size_t)(2 * c + (b0 >= lo ? 0 : 1)) * N * kTile + row;
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[j] = __fadd_rn(acc[j], __ldcg(theirs + j * kTile));
            if (c + 1 == (int)gridDim.x) break;
          }
        }
      }
      if (write && r < a.rows) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
          if (j < a.nb) st_out(a.y, a.ytype, (int64_t)j * a.ldy + r, acc[j] * a.out_scale);
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[j] = 0.0f;
      ++tile;
      k = 0;
    }
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
      for (int s = max(0, B.issued - kBuffers + 1); s <= B.issued; ++s)
        (void)mbar_wait_bounded(&B.done[s % kBuffers], (uint32_t)((s / kBuffers) & 1));
    }
    __syncthreads();
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == kMmaWarp)
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
const void* kernel_of(int nbt, bool fold) {
  if constexpr (BF16) {
    if (fold)
      return nbt == 1 ? (const void*)g4_kernel<true, 1, R, true>
             : nbt == 2 ? (const void*)g4_kernel<true, 2, R, true> : (const void*)g4_kernel<true, 4, R, true>;
  }
  switch (nbt) {
    case 1: return (const void*)g4_kernel<BF16, 1, R, false>;
    case 2: return (const void*)g4_kernel<BF16, 2, R, false>;
    case 4: return (const void*)g4_kernel<BF16, 4, R, false>;
    case 8: return (const void*)g4_kernel<BF16, 8, R, false>;
    case 16: return (const void*)g4_kernel<BF16, 16, R, false>;
  }
  if constexpr (R <= 2) {
    if (nbt == 32) return (const void*)g4_kernel<BF16, 32, R, false>;
  }
  if constexpr (R == 1) {
    if (nbt == 48) return (const void*)g4_kernel<BF16, 48, R, false>;
    if (nbt == 64) return (const void*)g4_kernel<BF16, 64, R, false>;
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
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;

  KernelArgs k{};
  k.scales = a.scales;
  k.mins = a.mins;
  k.s_ld = a.s_ld;
  k.rows = a.rows;
  k.group = a.group;
  k.lines = (a.cols + std::min(a.group, kHalf) - 1) / std::min(a.group, kHalf);
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
  k.steps = p.steps;
  k.wait_ns = a.wait_ns;
  k.status = a.status;
  const bool bf16 = a.xtype != NLS_DT_F16;
  const size_t xes = dt_size(a.xtype), yes = dt_size(a.ytype);
  for (int b0 = 0; b0 < a.nb; b0 += p.nmax) {
    k.nb = std::min(p.nmax, a.nb - b0);
    const int nbt = batch_of(k.nb), n = mma_n(nbt);
    k.y = static_cast<uint8_t*>(a.y) + (size_t)b0 * a.ldy * yes;
    const bool fold = folded(p.parts, k.nb);
    k.parts = fold ? 1 : p.parts;  // MMA passes over the columns
    k.x_off = kRawBytes;
    k.s_off = k.x_off + k.parts * n * kStep * 2;
    k.m_off = k.s_off + 2 * p.regions * kTile * k.ssize;
    k.stage_bytes = (k.m_off + (a.mins ? 2 * p.regions * kTile * k.ssize : 0) + 1023) & ~1023;
    const int room = 227 * 1024 - 1024 - (int)sizeof(Bars);
    k.stages = std::min(kMaxStages, room / k.stage_bytes);
    const size_t smem = (size_t)k.stages * k.stage_bytes + sizeof(Bars);
    const void* kern = p.regions == 4 ? (bf16 ? kernel_of<true, 4>(nbt, fold) : kernel_of<false, 4>(nbt, fold))
                       : p.regions == 2 ? (bf16 ? kernel_of<true, 2>(nbt, fold) : kernel_of<false, 2>(nbt, fold))
                                        : (bf16 ? kernel_of<true, 1>(nbt, fold) : kernel_of<false, 1>(nbt, fold));
    if (!kern) return cudaErrorInvalidValue;
    const void* x = static_cast<const uint8_t*>(a.x) + (size_t)b0 * a.ldx * xes;
    with_type(a.xtype, [&](auto xv) {
      using X = decltype(xv);
      g4_layout_kernel<X><<<2 * p.ksteps, 16 * n, 0, st>>>(static_cast<const X*>(x), a.ldx, k.nb, n, a.cols, p.parts,
                                                       fold ? nbt : 0, p.regions, ws, const_cast<float*>(k.xsum), k.count, p.tiles,
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
