// Values of the three types and 32-bit registers: conversions one and two at a time, packed 32-bit arithmetic, sums over a
// warp.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "block_ops.h"

namespace pccl {
namespace block {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
// One rounding to nearest even from 32 bits.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two neighbours, as they lie in a 32-bit word.
__device__ __forceinline__ void unpack2(uint32_t w, float* f, __nv_bfloat16) {
  f[0] = __uint_as_float(w << 16);
  f[1] = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, float* f, __half) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
  f[0] = v.x;
  f[1] = v.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Two 32-bit operations an instruction (sm_100), each rounded like its scalar form.
__device__ __forceinline__ uint64_t bits_of(float2 v) { return *reinterpret_cast<uint64_t*>(&v); }
__device__ __forceinline__ float2 pair_of(uint64_t b) { return *reinterpret_cast<float2*>(&b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
  return pair_of(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)));
  return pair_of(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)));
  return pair_of(d);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace block
}  // namespace pccl

// Calls BODY with the type `T` that stands for a DType.
#define PCCL_BLOCK_TYPES(DTYPE, T, ...)                                                    \
  switch (DTYPE) {                                                                         \
    case ::pccl::block::DType::kF32: { using T = float; __VA_ARGS__; break; }              \
    case ::pccl::block::DType::kF16: { using T = __half; __VA_ARGS__; break; }             \
    case ::pccl::block::DType::kBF16: { using T = __nv_bfloat16; __VA_ARGS__; break; }     \
  }
