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

// Pairs of float32: one instruction for two additions, products or
// multiply-adds, each rounded as the single operation is.
__device__ __forceinline__ uint64_t per_bits(float2 a) {
  return (uint64_t)__float_as_uint(a.x) | ((uint64_t)__float_as_uint(a.y) << 32);
}
__device__ __forceinline__ float2 per_pair(uint64_t u) {
  return make_float2(__uint_as_float((uint32_t)u), __uint_as_float((uint32_t)(u >> 32)));
}
__device__ __forceinline__ float2 per_both(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 per_add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(per_bits(a)), "l"(per_bits(b)));
  return per_pair(r);
}
__device__ __forceinline__ float2 per_mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(per_bits(a)), "l"(per_bits(b)));
  return per_pair(r);
}
__device__ __forceinline__ float2 per_fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(per_bits(a)), "l"(per_bits(b)), "l"(per_bits(c)));
  return per_pair(r);
}

// Two neighbouring 16-bit values in a 32-bit word (the first in the lower half),
// or one float32.
template <typename T>
__device__ __forceinline__ float2 per_unpack(uint32_t u);
template <>
__device__ __forceinline__ float2 per_unpack<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 per_unpack<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <typename T>
__device__ __forceinline__ uint32_t per_pack(float2 f);
template <>
__device__ __forceinline__ uint32_t per_pack<__nv_bfloat16>(float2 f) {
  const __nv_bfloat162 h = __float22bfloat162_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t per_pack<__half>(float2 f) {
  const __half2 h = __float22half2_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Pair i of the 16 bytes of a vector.
template <typename T>
__device__ __forceinline__ float2 per_pair_of(const uint4& u, int i) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (sizeof(T) == 4)
    return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  else
    return per_unpack<T>(w[i]);
}
template <typename T>
__device__ __forceinline__ void per_set_pair(uint4& u, int i, float2 f) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
  if constexpr (sizeof(T) == 4) {
    w[2 * i] = __float_as_uint(f.x);
    w[2 * i + 1] = __float_as_uint(f.y);
  } else {
    w[i] = per_pack<T>(f);
  }
}

static inline int64_t per_dtype_bytes(int32_t dtype) {
  return dtype == PER_F32 ? 4 : dtype == PER_BF16 || dtype == PER_F16 ? 2 : 0;
}
