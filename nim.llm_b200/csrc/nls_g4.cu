// nls_g4.cu -- nls_g4_matmul: y[b][r] = sum_c w(r, c) x[b][c] for 4-bit
// weights with a scale (and minimum) per group of columns.
//
// With q' = q - 8 and, where there are minimums, m' = m + 8 s:
//   y[b][r] = sum_g ( s[g][r] * sum_{c in g} q'[r][c] x[b][c]
//                     + m'[g][r] * sum_{c in g} x[b][c] )
// One warp per weight row: a lane takes the eight values of a 32-bit word,
// every 32nd word of the row; a group's terms are scaled as they are added.
// fp32 and bfloat16 activations enter as x 2^-12, and the result is multiplied
// by 2^12: 128 products with q' reach 2^10 times the largest activation, which
// would pass fp32's range before the scales bring it down.
#include <type_traits>

#include "nls_kernels.h"
#include "nls_types.cuh"

namespace nls {

namespace {

constexpr int kWarps = 8;
constexpr int kBatch = 8;

template <class X, class S, class Y>
__global__ void __launch_bounds__(32 * kWarps) g4_kernel(const G4Args a) {
  const int r = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.status = NLS_OK;
  if (r >= a.rows) return;
  const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.q) + (int64_t)r * a.q_ld);
  const S* sc = static_cast<const S*>(a.scales);
  const S* mn = static_cast<const S*>(a.mins);
  const X* x = static_cast<const X*>(a.x);
  Y* y = static_cast<Y*>(a.y);
  constexpr bool kShift = !std::is_same<X, __half>::value;
  constexpr float kIn = kShift ? 0x1p-12f : 1.0f, kOut = kShift ? 0x1p12f : 1.0f;
  for (int b0 = 0; b0 < a.nb; b0 += kBatch) {
    float acc[kBatch] = {};
    for (int i = lane; i < a.cols / 8; i += 32) {
      const uint32_t w = q[i];
      const int64_t g = (8 * i) / a.group;
      const float s = to_f32(sc[g * a.s_ld + r]);
      const float m = mn ? to_f32(mn[g * a.s_ld + r]) + 8.0f * s : 0.0f;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (b0 + b >= a.nb) break;
        const X* xb = x + (int64_t)(b0 + b) * a.ldx + 8 * i;
        float dot = 0.0f, sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = to_f32(xb[e]) * kIn;
          dot = fmaf((float)((int)((w >> (4 * e)) & 15u) - 8), v, dot);
          sum += v;
        }
        acc[b] = fmaf(s, dot, acc[b]);
        if (mn) acc[b] = fmaf(m, sum, acc[b]);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      for (int o = 16; o > 0; o >>= 1) acc[b] += __shfl_xor_sync(0xffffffffu, acc[b], o);
      if (lane == 0 && b0 + b < a.nb) y[(int64_t)(b0 + b) * a.ldy + r] = from_f32<Y>(acc[b] * kOut);
    }
  }
}

}  // namespace

size_t g4_workspace_bytes(const G4Args&, int) { return 0; }

cudaError_t launch_g4(const G4Args& a, void*, int, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.rows + kWarps - 1) / kWarps);
  with_type(a.xtype, [&](auto xv) {
    with_type(a.stype, [&](auto sv) {
      with_type(a.ytype, [&](auto yv) {
        g4_kernel<decltype(xv), decltype(sv), decltype(yv)><<<grid, 32 * kWarps, 0, st>>>(a);
      });
    });
  });
  return cudaGetLastError();
}

}  // namespace nls
