// Element types of the learner's operators (PER_F32 / PER_BF16 / PER_F16):
// arithmetic is float32, a 16-bit value is rounded once (to nearest even) on
// its way out.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

__device__ __forceinline__ float per_to_f32(float v) { return v; }
__device__ __forceinline__ float per_to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float per_to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T per_from_f32(float v);
template <>
__device__ __forceinline__ float per_from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 per_from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half per_from_f32<__half>(float v) {
  return __float2half_rn(v);
}

static inline int64_t per_dtype_bytes(int32_t dtype) {
  return dtype == PER_F32 ? 4 : dtype == PER_BF16 || dtype == PER_F16 ? 2 : 0;
}
