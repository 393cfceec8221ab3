// Shared device helpers of the token operators (layer norm, gated
// feed-forward, dropout): element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ccv_b200.h"

namespace ccv {

// Every operator computes in fp32; a 16-bit value is widened exactly on load
// and rounded (to nearest, ties to even) once on store.
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

template <typename T>
constexpr bool kIsBf16 = false;
template <>
constexpr bool kIsBf16<__nv_bfloat16> = true;

inline size_t dtype_bytes(int dtype) { return dtype == CCV_DTYPE_F32 ? 4 : 2; }
inline bool valid_dtype(int dtype) {
  return dtype == CCV_DTYPE_F32 || dtype == CCV_DTYPE_BF16 || dtype == CCV_DTYPE_F16;
}

}  // namespace ccv
