// nls_g4.cu -- nls_g4_matmul: y[b][r] = sum_c w(r, c) x[b][c] for 4-bit
// weights with a scale (and minimum) per group of columns, on the 5th-
// generation tensor cores.
//
// With q' = q - 8 and, where there are minimums, m' = m + 8 s:
//   y[b][r] = sum_g ( s[g][r] * sum_{c in g} q'[r][c] x[b][c]
//                     + m'[g][r] * sum_{c in g} x[b][c] )
// The inner sums are formed by the tensor cores without rounding a weight, the
// scales stay outside them in fp32. Two ways:
//  * Integers (few batch rows). The activations of a row's 128 columns are
//    fixed-point numbers X 2^-e of 31 bits (the largest has 30, so what is cut
//    off is 2^-31 of it), split into four signed bytes, which are four columns
//    of a tcgen05.mma kind::i8 against the nibbles themselves as unsigned
//    bytes: every product and sum is exact. 8 sum(X) is taken off afterwards,
//    in integers, and the four sums joined in fp32. Two or three logical
//    operations unpack 8 weights.
//  * Floating point (more batch rows: one column each instead of four). q' is
//    exact in fp16 and bfloat16; kind::f16 sums exact products in fp32. fp32
//    activations are split into three bfloat16 parts that hold all 24 bits,
//    multiplied one after the other into the same accumulator. fp32 and
//    bfloat16 activations enter as x 2^-12 and the result is multiplied by
//    2^12: 128 products with q' reach 2^10 times the largest activation, which
//    would pass fp32's range before the scales bring it down.
//
// What bounds it: at a few batch rows the weights' bytes (half a byte per
// weight); turning them into operands is the work per byte. So the A operand
// never touches shared memory: a thread owns a weight row, reads its packed
// bytes from the staged tile, unpacks them in registers and stores them to
// tensor memory (tcgen05.st), from where the MMA reads A; the sums come back to
// a thread of the same row (tcgen05.ld), whose scale is one register. The K
// order inside a word is the unpacking's; the activations are laid out in that
// order once per call. Unpacking to 16 bits (4 logical operations, 1-3 shifts
// and 4 packed subtractions per 8 weights, and 4 bytes per packed byte into
// tensor memory) holds the floating-point way to two thirds of the rate of the
// integer one at one row. Measured (128256 x 4096, groups of 128, bfloat16: 271
// MB of weights and scales, 42 us at the rate of a plain copy; captured calls one
// after the other): 1 / 4 / 12 batch rows 54 / 59 / 76 us (one row 5.0 TB/s), 16 /
// 32 / 64 rows 81 / 94 / 122 us. More rows read and unpack the weights again for
// every 64 of them (128 rows 244 us), with groups of 64 or fp32 activations for
// every 32, with groups of 32 for every 16 (151936 x 4096: 16 / 32 / 64 rows 138 /
// 272 / 543 us). About 10 us of each call are outside the stream: two launches,
// the pipeline's filling and the joining of split tiles.
//
// Work: a tile is 256 weight rows (two MMAs of M = 128), a step 256 columns of
// it: 128 bytes of a row, since the copy of a step costs the copy engine about
// 4 cycles a row however short the row (64-byte rows held the kernel to 3.4
// TB/s). The steps of all tiles, in order, are dealt out evenly to the CTAs (one
// per SM), so an SM's load is within one step of every other's whatever the
// shape; a tile that more than one CTA worked on is joined by the last of them
// to finish, from partial sums in the workspace added in CTA order (the same
// bits every time; no CTA waits for another).
// One CTA: 8 or 16 warps unpack (a thread its row's 256 columns, half after
// half, or one half of them), 8 or 16 add the halves' sums to their rows' (16:
// two sets, each one half of the batch rows), one issues the copies (a ring of
// stages: packed weights by tensor map, activations, scales) and one the MMAs. Roles only wait for one
// another through mbarriers, and each runs as far ahead as its buffers let it:
// operands have one buffer per half in TMEM, accumulators as many as fit in
// the rest.
#include <cuda.h>

#include <algorithm>
#include <atomic>
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

constexpr int kRawBytes = kTile * kStep / 2;
constexpr int kMaxStages = 8;
constexpr uint32_t kTmemCols = 512;
constexpr int kMaxSmem = 227 * 1024;

enum class Op { kI8, kF16, kBF16 };
// Tensor memory: a half step's operand takes 32 (bytes) or 64 columns per tile
// half, two tile halves in each half step's buffer; the rest are accumulators
__host__ __device__ constexpr int a_cols(Op op) { return op == Op::kI8 ? 32 : 64; }
__host__ __device__ constexpr int acc_cols(Op op) { return (int)kTmemCols - 4 * a_cols(op); }

// The split of a CTA's warps, 24 for unpacking and adding at most (72 registers
// a thread). Unpacking bytes is cheap, and adding four sums per batch row is
// not: 8 and 16 (one batch row leaves nothing for a second set). Unpacking to
// 16 bits is the larger part up to 16 batch rows (81 us with 16 and 8, 87 with
// 8 and 16, on 128256 x 4096); above, adding is (32 rows: 95.5 and 94 us).
__host__ __device__ constexpr int unpack_warps(Op op, int nbt) { return op != Op::kI8 && nbt <= 16 ? 16 : 8; }
__host__ __device__ constexpr int add_warps(Op op, int nbt) {
  return op != Op::kI8 ? (nbt <= 16 ? 8 : 16) : nbt == 1 ? 8 : 16;
}
__host__ __device__ constexpr int threads_of(Op op, int nbt) { return 32 * (unpack_warps(op, nbt) + add_warps(op, nbt) + 2); }

// groups (scales) per half step
__host__ __device__ constexpr int regions_of(int group) { return group == 32 ? 4 : group == 64 ? 2 : 1; }
// batch rows a launch is compiled for, and the MMA's columns
__host__ __device__ constexpr int batch_of(Op op, int nb) {
  if (op == Op::kI8) return nb <= 1 ? 1 : nb <= 2 ? 2 : nb <= 4 ? 4 : nb <= 8 ? 8 : 12;
  return nb <= 8 ? 8 : nb <= 16 ? 16 : nb <= 32 ? 32 : nb <= 48 ? 48 : 64;
}
__host__ __device__ constexpr int mma_n(Op op, int nbt) {
  return op == Op::kI8 ? (nbt <= 4 ? 16 : 4 * nbt) : (nbt <= 16 ? 16 : nbt);
}
// The most batch rows the integer way takes. By tensor memory, two buffers of
// accumulators have to fit (96 columns per tile half and buffer): 4 rows with
// groups of 32, 12 with groups of 64. By the times, in integers and in floating
// point: wide groups, 128256 x 4096, 12 rows 76 and 81 us, 16 rows 106 and 81;
// groups of 64, 151936 x 4096, fp32 activations 5 to 8 rows 117 and 146 us, 9 to
// 12 138 and 149; 16-bit ones 117 and 92, 138 and 99 (1 to 4 rows in integers: 68
// to 85).
__host__ __device__ constexpr int i8_rows(int regions, bool f32) { return regions == 4 || (regions == 2 && !f32) ? 4 : 12; }
// bytes of a half step's laid-out activations: bytes (and per region and batch
// row four words for the joining), or 16-bit parts (and per region and column
// their sum)
__host__ __device__ constexpr int x_half(Op op, int nbt, int regions, int parts) {
  return op == Op::kI8 ? mma_n(op, nbt) * kHalf + regions * nbt * 16
                       : mma_n(op, nbt) * (parts * kHalf * 2 + regions * 4);
}

// How a launch of nb batch rows goes, `left` of the call's rows being left.
struct Way {
  Op op;
  int nb, nbt, n, parts;
};

Way way_of(const G4Args& a, int left) {
  Way w;
  const int regions = regions_of(a.group);
  w.op = left <= i8_rows(regions, a.xtype == NLS_DT_F32) ? Op::kI8 : a.xtype == NLS_DT_F16 ? Op::kF16 : Op::kBF16;
  w.parts = w.op != Op::kI8 && a.xtype == NLS_DT_F32 ? 3 : 1;
  // regions x N columns: 64 per tile half and buffer. (fp32's three parts: a
  // stage of 64 rows would leave room for one stage only)
  w.nb = w.op == Op::kI8 ? left : std::min(left, std::min(64 / regions, w.parts == 3 ? 32 : 64));
  w.nbt = batch_of(w.op, w.nb);
  w.n = mma_n(w.op, w.nbt);
  return w;
}

struct Plan {
  int ksteps, tiles, grid, regions;
  int64_t steps;  // tiles * ksteps
  // workspace
  size_t x_bytes, part_bytes, count_bytes;
  size_t total() const { return x_bytes + part_bytes + count_bytes; }
};

Plan plan_of(const G4Args& a, int sm_count) {
  Plan p{};
  p.ksteps = (a.cols + kStep - 1) / kStep;
  p.tiles = (a.rows + kTile - 1) / kTile;
  p.steps = (int64_t)p.tiles * p.ksteps;
  p.grid = (int)std::min<int64_t>(sm_count, p.steps);
  p.regions = regions_of(a.group);
  for (int b0 = 0; b0 < a.nb;) {
    const Way w = way_of(a, a.nb - b0);
    const size_t halves = (size_t)p.ksteps * 2;
    p.x_bytes = std::max(p.x_bytes, (halves * x_half(w.op, w.nbt, p.regions, w.parts) + 255) & ~size_t(255));
    p.part_bytes = std::max(p.part_bytes, (size_t)p.grid * 2 * w.nbt * kTile * sizeof(float));
    b0 += w.nb;
    if (a.nb - b0 > 2 * 64) b0 = a.nb - 64 - (a.nb - b0) % 64;  // (passes in between are all alike)
  }
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
  const uint8_t* x;     // laid-out activations, x_half bytes per half step
  float* part;          // partial tiles [2 * grid][NB][256]
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

// eight activations of a batch row as fp32 (past the matrix: zeros; columns come
// in whole 32)
template <class X>
__device__ __forceinline__ void load8(const X* x, int64_t ldx, int nb, int cols, int n, int c0, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.0f;
  if (n >= nb || c0 >= cols) return;
  const X* p = x + (int64_t)n * ldx + c0;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    X t[8];
#pragma unroll
    for (int e = 0; e < (int)(8 * sizeof(X) / 16); ++e) reinterpret_cast<uint4*>(t)[e] = reinterpret_cast<const uint4*>(p)[e];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32(t[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32(p[e]);
  }
}

__device__ __forceinline__ void clear_counts(int* count, int tiles, int* status, int clear_status) {
  const int i0 = (int)(blockIdx.x * blockDim.x + threadIdx.x);
  if (i0 == 0 && clear_status) *status = NLS_OK;
  for (int i = i0; i < tiles; i += (int)(gridDim.x * blockDim.x)) count[i] = 0;
}

// The integer way. One block per half step; the 16 threads of a batch row take 8
// columns each. Their largest magnitude gives the row's exponent there: X =
// x 2^e with |X| < 2^30 is exact but for the rounding to a whole number; its
// four bytes p0 2^24 + p1 2^16 + p2 2^8 + p3, each -128 .. 127, are columns 4 n
// .. 4 n + 3 of the operand (no-swizzle K-major: 8 rows x 16 bytes per core
// matrix, K step j of 32 columns at j * N * 32). Behind the operand, per
// region and batch row: 8 (sum p0 2^8 + sum p1), 8 (sum p2 2^8 + sum p3), 2^-e
// and sum X. A row with an infinity or a NaN has NaN for 2^-e. (The exponent
// stops at 2^-96: 2^-e stays a normal number; what that loses is below 2^-125.)
template <class X>
__global__ void __launch_bounds__(512) g4_bytes_kernel(const X* x, int64_t ldx, int nb, int nbt, int n_cols, int cols,
                                                       int regions, uint8_t* op, int half_bytes, int* count, int tiles,
                                                       int* status, int clear_status) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  clear_counts(count, tiles, status, clear_status);
  const int k = blockIdx.x, n = threadIdx.x >> 4, word = threadIdx.x & 15;
  float v[8];
  load8(x, ldx, nb, cols, n, k * kHalf + word * 8, v);
  float top = 0.0f;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top = fmaxf(top, fabsf(v[e]));
    bad |= !isfinite(v[e]);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
  }
  // top < 2^(E + 1), E the exponent field's: X below 2^30
  const int E = max((int)(__float_as_uint(top) >> 23) - 127, -96);
  const double up = __longlong_as_double((long long)(29 - E + 1023) << 52);
  int sum[4] = {0, 0, 0, 0};
  uint32_t lo[4] = {0u, 0u, 0u, 0u}, hi[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    int f = bad ? 0 : __double2int_rn((double)v[e] * up);
#pragma unroll
    for (int p = 3; p >= 0; --p) {
      const int d = (int)(int8_t)(f & 0xFF);
      f = (f - d) >> 8;
      sum[p] += d;
      // K order of a word: columns 0 2 4 6, then 1 3 5 7
      if (e & 1) hi[p] |= ((uint32_t)d & 0xFFu) << (4 * (e & 6));
      else lo[p] |= ((uint32_t)d & 0xFFu) << (4 * (e & 6));
    }
  }
  uint8_t* half = op + (size_t)k * half_bytes;
  uint8_t* dst = half + (word >> 2) * (n_cols * 32) + ((word >> 1) & 1) * 128 + (word & 1) * 8;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int c = 4 * n + p;
    *reinterpret_cast<uint2*>(dst + (c >> 3) * 256 + (c & 7) * 16) = make_uint2(lo[p], hi[p]);
  }
  const int lanes = 16 / regions;
  for (int o = 1; o < lanes; o <<= 1) {
#pragma unroll
    for (int p = 0; p < 4; ++p) sum[p] += __shfl_xor_sync(0xffffffffu, sum[p], o);
  }
  if (word % lanes == 0 && n < nbt) {
    const int a01 = sum[0] * 256 + sum[1], a23 = sum[2] * 256 + sum[3];
    const float unit = bad ? __int_as_float(0x7fffffff) : __uint_as_float((uint32_t)(E - 29 + 127) << 23);
    *reinterpret_cast<int4*>(half + n_cols * kHalf + ((word / lanes) * nbt + n) * 16) =
        make_int4(8 * a01, 8 * a23, __float_as_int(unit),
                  __float_as_int((float)((double)a01 * 65536.0 + (double)a23)));
  }
}

// The floating-point way. One block per half step; a thread takes 8 columns of a
// batch row and writes them, permuted, as one 16-byte line of the operand (no-
// swizzle K-major: 8 rows x 16 bytes per core matrix, K step j of 16 columns at
// j * N * 32), for each part.
// Behind the operand come their sums per region (the 16 threads of a batch row
// are neighbours). Rows nb .. N - 1 and columns past the matrix are zeros.
template <class X>
__global__ void __launch_bounds__(1024) g4_layout_kernel(const X* x, int64_t ldx, int nb, int n_cols, int cols,
                                                         int parts, int regions, uint8_t* op, int half_bytes, int* count,
                                                          int tiles, int* status, int clear_status) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  clear_counts(count, tiles, status, clear_status);
  const int k = blockIdx.x, n = threadIdx.x >> 4, word = threadIdx.x & 15;
  constexpr bool kF32 = std::is_same<X, float>::value;
  constexpr float kIn = std::is_same<X, __half>::value ? 1.0f : 0x1p-12f;
  float v[8];
  load8(x, ldx, nb, cols, n, k * kHalf + word * 8, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= kIn;
  uint8_t* half = op + (size_t)k * half_bytes;
  {
    float s = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    const int lanes = 16 / regions;
    for (int o = 1; o < lanes; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (word % lanes == 0)
      reinterpret_cast<float*>(half + parts * n_cols * (kHalf * 2))[(word / lanes) * n_cols + n] = s;
  }
  constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};
  uint8_t* dst = half + (size_t)(word >> 1) * (n_cols * 32) + (n >> 3) * 256 + (word & 1) * 128 + (n & 7) * 16;
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
    *reinterpret_cast<uint4*>(dst + (size_t)part * n_cols * (kHalf * 2)) = make_uint4(w[0], w[1], w[2], w[3]);
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
template <bool I8, bool ACC>
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t leader) {
  if constexpr (I8) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %4, 0;\n\t"
        "setp.ne.u32 p, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(leader), "n"(ACC ? 1 : 0)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %4, 0;\n\t"
        "setp.ne.u32 p, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(leader), "n"(ACC ? 1 : 0)
        : "memory");
  }
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

// The eight weights of a word, low nibble first. Floating point: q - 8 in pairs
// (0, 4) (1, 5) (2, 6) (3, 7):
// a nibble under the exponent of 2^10 (fp16) or 2^7 (bfloat16) is that power
// plus q, exactly; fp16's 10 bits of mantissa take the nibble at bit 4 too, as
// 2^10 + 16 q.
template <bool BF16>
struct UnpackF {
  // the power of two's bits, out of the compiler's sight: as an immediate it
  // would take a logical operation of its own beside the mask's
  uint32_t magic;
  __device__ __forceinline__ UnpackF() { asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(BF16 ? 0x43004300 : 0x64006400)); }
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

// Integers: q as bytes 0 2 4 6, then 1 3 5 7.
struct UnpackI {
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t* o) const {
    o[0] = w & 0x0F0F0F0Fu;
    o[1] = (w >> 4) & 0x0F0F0F0Fu;
  }
};
template <Op OP>
struct UnpackOf {
  using type = UnpackF<OP == Op::kBF16>;
};
template <>
struct UnpackOf<Op::kI8> {
  using type = UnpackI;
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
  uint64_t ready[2];            // a half's operand is stored
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

// NB: batch rows. R: groups per half step.
template <Op OP, int NB, int R>
__global__ void __launch_bounds__(threads_of(OP, NB), 1)
    g4_kernel(const KernelArgs a, const __grid_constant__ CUtensorMap qmap) {
  constexpr bool I8 = OP == Op::kI8;
  constexpr int N = mma_n(OP, NB);
  constexpr int kACols = a_cols(OP);                // of a tile half's operand
  constexpr uint32_t kTmemD = 4 * kACols;           // the accumulators' first column
  constexpr int kFit = acc_cols(OP) / (2 * R * N) & ~1;
  constexpr int kBuffers = kFit < kMaxBuffers ? kFit : kMaxBuffers;
  constexpr int kMmas = I8 ? 4 : 8;                 // per tile half and half step: K = 32 or 16
  constexpr int kUnpackWarps = unpack_warps(OP, NB), kAddWarps = add_warps(OP, NB);
  constexpr int kCopyWarp = kUnpackWarps + kAddWarps, kMmaWarp = kCopyWarp + 1;
  constexpr int CB = NB * 8 / kAddWarps < 1 ? 1 : NB * 8 / kAddWarps;  // batch rows per adding thread
  // A step's two halves are added together where that leaves the MMAs another
  // step's accumulators (the waits and loads of a step are then one chain)
  constexpr int kTogether = kBuffers >= 4 ? 2 : 1;
  static_assert(NB * (I8 ? 4 : 1) <= N && kBuffers >= 2, "columns");
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
    for (int i = 0; i < 2; ++i) mbar_init(&B.ready[i], 8);
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
  // the laid-out activations and the cleared counters are there
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
      const uint32_t xb = (uint32_t)(2 * x_half(OP, NB, R, a.parts));
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
    // s32 += u8 x s8, or f32 += f16 x f16 (bf16 x bf16); both K-major
    constexpr uint32_t kBF = OP == Op::kBF16 ? 1u : 0u;
    constexpr uint32_t idesc = (I8 ? (2u << 4) | (1u << 10) : (1u << 4) | (kBF << 7) | (kBF << 10)) |
                               ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    // no-swizzle K-major descriptor: 128 bytes from a row's first 16 bytes to
    // its next 16, 256 from 8 rows to the next
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
        const uint64_t bd = bd0 + (uint64_t)(slot.i * (a.stage_bytes >> 4) + h * (x_half(OP, NB, R, a.parts) >> 4));
        const uint32_t ab = tbase + (uint32_t)(h * 2 * kACols), db = tbase + kTmemD + (uint32_t)(buf.i * (2 * R * N));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int j = 0; j < kMmas; ++j) {
            const uint32_t d = db + (t * R + j * R / kMmas) * N, A = ab + t * kACols + 8 * j;
            if (j % (kMmas / R) == 0) mma<I8, false>(d, A, bd + j * (N * 2), idesc, leader);
            else mma<I8, true>(d, A, bd + j * (N * 2), idesc, leader);
          }
        }
        if constexpr (OP == Op::kBF16) {
          for (int p = 1; p < a.parts; ++p) {
            const uint64_t bp = bd + (uint64_t)(p * kMmas * N * 2);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int j = 0; j < kMmas; ++j)
                mma<I8, true>(db + (t * R + j * R / kMmas) * N, ab + t * kACols + 8 * j, bp + j * (N * 2), idesc, leader);
          }
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
    const int quarter = warp & 3, t = (warp >> 2) & 1;
    const int row = t * 128 + quarter * 32 + lane;  // in the tile
    constexpr int kMine = 16 / kUnpackWarps;        // halves of a step it unpacks, from h1 on
    const int h1 = kMine == 2 ? 0 : warp >> 3;
    const uint32_t ta = tbase + ((uint32_t)(32 * quarter) << 16) + (uint32_t)(t * kACols);
    // 16-byte pieces of a 128-byte row lie where the 128-byte swizzle of the
    // copy put them (free of bank conflicts); the second half's 64 bytes on
    uint32_t at[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) at[c] = sbase + (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4)) ^ (uint32_t)(h1 << 6);
    const typename UnpackOf<OP>::type unpack{};
    constexpr int kWords = kACols / 16;         // operand words per packed word
    constexpr int kPieces = 32 / (4 * kWords);  // 16-byte pieces per store of 32 words
    Ring slot{0, 0}, prev{h1, 0};  // stage; accumulators of the half a step before
    for (int s = 0; s < nsteps && !fail; ++s) {
      if (!warp_wait(full0 + (uint32_t)slot.i * 8, slot.phase, a.wait_ns)) {
        fail = true;
        break;
      }
      const uint32_t st = (uint32_t)(slot.i * a.stage_bytes);
      slot.next(a.stages);
#pragma unroll
      for (int h = 0; h < kMine; ++h) {
#pragma unroll
        for (int i = 0; i < kACols / 32; ++i) {
          uint32_t o[32];
#pragma unroll
          for (int c = 0; c < kPieces; ++c) {
            uint32_t v[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                         : "r"((at[kPieces * i + c] ^ (uint32_t)(h << 6)) + st)
                         : "memory");
#pragma unroll
            for (int e = 0; e < 4; ++e) unpack(v[e], o + (4 * c + e) * kWords);
          }
          // the step before had the same operand buffer
          if (i == 0 && s >= 1) {
            if (!warp_wait(done0 + (uint32_t)prev.i * 8, prev.phase, a.wait_ns)) {
              fail = true;
              break;
            }
            prev.next(kBuffers, 2 / kMine);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
          tmem_st32(ta + (uint32_t)((h1 + h) * 2 * kACols + i * 32), o);
        }
        if (fail) break;
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(ready0 + (uint32_t)(h1 + h) * 8);
      }
    }
  } else {
    const int aw = warp - kUnpackWarps, quarter = aw & 3, t = (aw >> 2) & 1, set = aw >> 3;
    const int row = t * 128 + quarter * 32 + lane;  // in the tile
    const int b0 = set * CB;                        // its first batch row
    const uint32_t td = tbase + ((uint32_t)(32 * quarter) << 16) + kTmemD + (uint32_t)(t * R * N + b0 * (I8 ? 4 : 1));
    float acc[CB];
#pragma unroll
    for (int j = 0; j < CB; ++j) acc[j] = 0.0f;
    int ends = 0;              // tiles joined so far (phase of the joining barriers)
    int tile = tile0, k = k0;  // position of the step
    Ring slot{0, 0}, buf{0, 0};
    for (int s = 0; s < nsteps; ++s) {
      const uint8_t* st = smem + (uint32_t)(slot.i * a.stage_bytes);
#pragma unroll 1
      for (int h0 = 0; h0 < 2; h0 += kTogether) {
        // the scales have landed with the stage
        if (h0 == 0 && !warp_wait(full0 + (uint32_t)slot.i * 8, slot.phase, a.wait_ns)) {
          fail = true;
          break;
        }
        float sc[kTogether][R], mn[kTogether][R];
#pragma unroll
        for (int h = 0; h < kTogether; ++h)
#pragma unroll
          for (int r = 0; r < R; ++r) {  // (the last step may have fewer)
            const int l = (h0 + h) * R + r;
            const bool in = 2 * k * R + l < a.lines;
            sc[h][r] = in ? ld_scale(st + a.s_off, a.stype, l * kTile + row) : 0.0f;
            mn[h][r] = in && a.mins ? __fmaf_rn(8.0f, sc[h][r], ld_scale(st + a.m_off, a.stype, l * kTile + row)) : 0.0f;
          }
        // (the MMAs of the second half complete after the first's)
        if (!warp_wait(done0 + (uint32_t)(buf.i + kTogether - 1) * 8, buf.phase, a.wait_ns)) {
          fail = true;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // batch rows per load: at most 32 words of sums at a time
        constexpr int kWordsPer = (I8 ? 4 : 1) * R * kTogether;
        constexpr int kMost = 32 / kWordsPer < (I8 ? 2 : 8) ? 32 / kWordsPer : (I8 ? 2 : 8);
        constexpr int C = CB < kMost ? CB : kMost;
        static_assert(CB % C == 0, "batch rows per load");
#pragma unroll
        for (int c = 0; c < CB; c += C) {
          uint32_t d[kTogether][R][C * (I8 ? 4 : 1)];
#pragma unroll
          for (int h = 0; h < kTogether; ++h)
#pragma unroll
            for (int r = 0; r < R; ++r)
              tmem_ld<C * (I8 ? 4 : 1)>(td + (uint32_t)((buf.i + h) * (2 * R * N) + r * N + c * (I8 ? 4 : 1)), d[h][r]);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          if (c + C >= CB) {  // all sums are in registers: the MMAs may have their place
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
#pragma unroll
              for (int h = 0; h < kTogether; ++h) arrive(added0 + (uint32_t)(buf.i + h) * 8);
            }
          }
#pragma unroll
          for (int h = 0; h < kTogether; ++h)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int j = 0; j < C; ++j) {
                if constexpr (I8) {
                  // sum (q - 8) X: each pair of bytes' sums joined as integers
                  // (below 2^26 in magnitude), the pairs in fp32
                  const int4 e = *reinterpret_cast<const int4*>(st + a.x_off + (h0 + h) * x_half(OP, NB, R, 1) +
                                                                N * kHalf + (r * NB + b0 + c + j) * 16);
                  const uint32_t* p = d[h][r] + 4 * j;
                  const int hi = (int)(p[0] * 256u + p[1]) - e.x, lo = (int)(p[2] * 256u + p[3]) - e.y;
                  float f = __fmul_rn(sc[h][r], __fmaf_rn(__int2float_rn(hi), 65536.0f, __int2float_rn(lo)));
                  if (a.mins) f = __fmaf_rn(mn[h][r], __int_as_float(e.w), f);
                  acc[c + j] = __fmaf_rn(f, __int_as_float(e.z), acc[c + j]);
                } else {
                  acc[c + j] = __fmaf_rn(sc[h][r], __uint_as_float(d[h][r][j]), acc[c + j]);
                }
              }
        }
        if (!I8 && a.mins) {
#pragma unroll
          for (int h = 0; h < kTogether; ++h) {
            const float* xs = reinterpret_cast<const float*>(st + a.x_off + (h0 + h) * x_half(OP, NB, R, a.parts) +
                                                             a.parts * (N * kHalf * 2)) + b0;
#pragma unroll
            for (int r = 0; r < R; ++r)  // (past the matrix: zero times a sum of zeros)
#pragma unroll
              for (int j = 0; j < CB; j += 4) {
                const float4 x4 = *reinterpret_cast<const float4*>(xs + r * N + j);
                acc[j] = __fmaf_rn(mn[h][r], x4.x, acc[j]);
                acc[j + 1] = __fmaf_rn(mn[h][r], x4.y, acc[j + 1]);
                acc[j + 2] = __fmaf_rn(mn[h][r], x4.z, acc[j + 2]);
                acc[j + 3] = __fmaf_rn(mn[h][r], x4.w, acc[j + 3]);
              }
          }
        }
        if (h0 + kTogether == 2) {
          __syncwarp();
          if (lane == 0) arrive(free0 + (uint32_t)slot.i * 8);
        }
        buf.next(kBuffers, kTogether);
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
        float* mine = a.part + (size_t)(2 * blockIdx.x + (tile == tile0 ? 0 : 1)) * NB * kTile + (size_t)b0 * kTile + row;
#pragma unroll
        for (int j = 0; j < CB; ++j) __stcg(mine + j * kTile, acc[j]);
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
          const int c0 = (int)(((lo + 1) * gridDim.x - 1) / a.steps);
          const int c1 = (int)(((lo + a.ksteps) * gridDim.x - 1) / a.steps);
          // (only the first's steps can begin before the tile; the loads of
          // several are in flight together)
          const float* theirs = a.part + ((size_t)(2 * c0) * NB + b0) * kTile + row;
          if (a.steps * c0 / gridDim.x < lo) theirs += NB * kTile;
#pragma unroll
          for (int j = 0; j < CB; ++j) acc[j] = __ldcg(theirs + j * kTile);
          constexpr int U = CB <= 2 ? 8 : CB <= 8 ? 4 : 1;
          for (int c = c0 + 1; c <= c1; c += U) {
            float v[U][CB];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int j = 0; j < CB; ++j)
                v[u][j] = c + u <= c1 ? __ldcg(a.part + ((size_t)(2 * (c + u)) * NB + b0 + j) * kTile + row) : 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int j = 0; j < CB; ++j)
                if (c + u <= c1) acc[j] = __fadd_rn(acc[j], v[u][j]);
          }
        }
      }
      if (write && r < a.rows) {
#pragma unroll
        for (int j = 0; j < CB; ++j)
          if (b0 + j < a.nb) st_out(a.y, a.ytype, (int64_t)(b0 + j) * a.ldy + r, acc[j] * a.out_scale);
      }
#pragma unroll
      for (int j = 0; j < CB; ++j) acc[j] = 0.0f;
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


// The kernels' dynamic shared memory limit, raised once per device to the most
// there is (the attribute call costs host time on every launch otherwise).
cudaError_t allow_smem(const void* kern, int bytes) {
  struct Seen {
    std::atomic<const void*> kern{nullptr};
    std::atomic<uint64_t> devices{0};
  };
  static Seen seen[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  for (Seen& k : seen) {
    const void* none = nullptr;
    if (k.kern.load(std::memory_order_acquire) != kern && !k.kern.compare_exchange_strong(none, kern) && none != kern)
      continue;
    if (dev < 64 && (k.devices.load(std::memory_order_acquire) >> dev & 1)) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    if (e == cudaSuccess && dev < 64) k.devices.fetch_or(1ull << dev, std::memory_order_release);
    return e;
  }
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <Op OP, int R>
const void* kernel_of(int nbt) {
  if constexpr (OP == Op::kI8) {
    switch (nbt) {
      case 1: return (const void*)g4_kernel<OP, 1, R>;
      case 2: return (const void*)g4_kernel<OP, 2, R>;
      case 4: return (const void*)g4_kernel<OP, 4, R>;
    }
    if constexpr (i8_rows(R, true) >= 12) {
      if (nbt == 8) return (const void*)g4_kernel<OP, 8, R>;
      if (nbt == 12) return (const void*)g4_kernel<OP, 12, R>;
    }
  } else {
    // (fewer rows than these are the integer way's)
    if constexpr (i8_rows(R, false) < 8) {
      if (nbt == 8) return (const void*)g4_kernel<OP, 8, R>;
    }
    if (nbt == 16) return (const void*)g4_kernel<OP, 16, R>;
    if constexpr (R <= 2) {
      if (nbt == 32) return (const void*)g4_kernel<OP, 32, R>;
    }
    if constexpr (R == 1) {
      if (nbt == 48) return (const void*)g4_kernel<OP, 48, R>;
      if (nbt == 64) return (const void*)g4_kernel<OP, 64, R>;
    }
  }
  return nullptr;
}
template <Op OP>
const void* kernel_of(int regions, int nbt) {
  return regions == 4 ? kernel_of<OP, 4>(nbt) : regions == 2 ? kernel_of<OP, 2>(nbt) : kernel_of<OP, 1>(nbt);
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
  k.part = reinterpret_cast<float*>(ws + p.x_bytes);
  k.count = reinterpret_cast<int*>(ws + p.x_bytes + p.part_bytes);
  k.ytype = a.ytype;
  k.ldy = a.ldy;
  k.ksteps = p.ksteps;
  k.steps = p.steps;
  k.wait_ns = a.wait_ns;
  k.status = a.status;
  const size_t xes = dt_size(a.xtype), yes = dt_size(a.ytype);
  for (int b0 = 0; b0 < a.nb;) {
    const Way w = way_of(a, a.nb - b0);
    const bool i8 = w.op == Op::kI8;
    const int half_bytes = x_half(w.op, w.nbt, p.regions, w.parts);
    k.nb = w.nb;
    k.parts = w.parts;
    k.out_scale = w.op == Op::kBF16 ? 4096.0f : 1.0f;
    k.y = static_cast<uint8_t*>(a.y) + (size_t)b0 * a.ldy * yes;
    k.x_off = kRawBytes;
    k.s_off = k.x_off + 2 * half_bytes;
    k.m_off = k.s_off + 2 * p.regions * kTile * k.ssize;
    k.stage_bytes = (k.m_off + (a.mins ? 2 * p.regions * kTile * k.ssize : 0) + 1023) & ~1023;
    const int room = kMaxSmem - 1024 - (int)sizeof(Bars);
    k.stages = std::min(kMaxStages, room / k.stage_bytes);
    const size_t smem = (size_t)k.stages * k.stage_bytes + sizeof(Bars);
    const void* kern = i8 ? kernel_of<Op::kI8>(p.regions, w.nbt)
                       : w.op == Op::kF16 ? kernel_of<Op::kF16>(p.regions, w.nbt)
                                          : kernel_of<Op::kBF16>(p.regions, w.nbt);
    if (!kern) return cudaErrorInvalidValue;
    const void* x = static_cast<const uint8_t*>(a.x) + (size_t)b0 * a.ldx * xes;
    const int clear = b0 == 0 ? 1 : 0;
    with_type(a.xtype, [&](auto xv) {
      using X = decltype(xv);
      if (i8)
        g4_bytes_kernel<X><<<2 * p.ksteps, 4 * w.n, 0, st>>>(static_cast<const X*>(x), a.ldx, w.nb, w.nbt, w.n, a.cols,
                                                             p.regions, ws, half_bytes, k.count, p.tiles, a.status,
                                                             clear);
      else
        g4_layout_kernel<X><<<2 * p.ksteps, 16 * w.n, 0, st>>>(static_cast<const X*>(x), a.ldx, w.nb, w.n, a.cols,
                                                               w.parts, p.regions, ws, half_bytes, k.count, p.tiles,
                                                               a.status, clear);
    });
    b0 += w.nb;
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    e = allow_smem(kern, (int)smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid, 1, 1);
    cfg.blockDim = dim3((unsigned)threads_of(w.op, w.nbt), 1, 1);
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
