// nls_types.cuh -- the element types of nls_g4_matmul and nls_draw_batch
// (NLS_DT_*): the C++ type of each and its conversions to and from fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstddef>
#include <cstdint>

#include "nimllm_sample.h"

namespace nls {

inline bool dt_ok(int dt) { return dt == NLS_DT_F32 || dt == NLS_DT_F16 || dt == NLS_DT_BF16; }
inline size_t dt_size(int dt) { return dt == NLS_DT_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// f(T{}) for the C++ type of an element type (checked by the caller)
template <class F>
auto with_type(int dt, F&& f) {
  switch (dt) {
    case NLS_DT_F16: return f(__half{});
    case NLS_DT_BF16: return f(__nv_bfloat16{});
    default: return f(float{});
  }
}

}  // namespace nls
