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

// V adjacent elements, moved by loads and stores of up to 16 bytes (the
// address is aligned to the smaller of 16 bytes and the whole).
template <typename T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Vec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.e[i] = from_f32<T>(f[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = v;
}

// Whether rows of `n` elements starting at p, `stride` apart, can be read
// V elements at a time.
template <typename T, int V>
inline bool vec_rows(const void* p, int64_t stride, int64_t n) {
  constexpr uintptr_t bytes = V * sizeof(T) < 16 ? V * sizeof(T) : 16;
  return n % V == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0 &&
         (static_cast<uint64_t>(stride) * sizeof(T)) % bytes == 0;
}

template <typename T>
constexpr bool kIsBf16 = false;
template <>
constexpr bool kIsBf16<__nv_bfloat16> = true;

inline size_t dtype_bytes(int dtype) { return dtype == CCV_DTYPE_F32 ? 4 : 2; }
inline bool valid_dtype(int dtype) {
  return dtype == CCV_DTYPE_F32 || dtype == CCV_DTYPE_BF16 || dtype == CCV_DTYPE_F16;
}

}  // namespace ccv
