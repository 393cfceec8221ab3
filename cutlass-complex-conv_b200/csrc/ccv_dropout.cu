// Dropout from a counter-based generator, with an optional residual added.
//
// Element i of a call with key `seed` and stream `offset` takes 16 bits of
// Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011) at counter (i / 8, offset): eight
// 16-bit parts per evaluation, low half of each word first.  It is dropped
// when its part is below t = round(p 65536), else scaled by 65536/(65536-t),
// the inverse of the share kept exactly, so the expectation is unbiased.
// The mask is a function of (seed, offset, i): the backward pass is the same
// kernel on the gradient, from the output's type to the input's, and nothing
// is stored.  Bound by memory with a
// residual (51 M elements, bf16 plus fp32: 80-84 us, 6.2-6.4 TB/s, 96-99 % of
// the copy rate on B200) and nearly so by the generator's issue slots without
// (25 M bf16: 19 us, 5.3 TB/s).  A gradient from one type to another, 51 M
// elements through autograd: fp32 to bf16 53 us, bf16 to fp32 64 us (308 MB).
#include <cmath>

#include "ccv_internal.h"
#include "ccv_ptx.cuh"
#include "ccv_tokens.cuh"

namespace ccv {

namespace {

__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint2 k) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c.x) * 0xD2511F53u;
    const uint64_t b = static_cast<uint64_t>(c.z) * 0xCD9E8D57u;
    c = make_uint4(static_cast<uint32_t>(b >> 32) ^ c.y ^ k.x, static_cast<uint32_t>(b),
                   static_cast<uint32_t>(a >> 32) ^ c.w ^ k.y, static_cast<uint32_t>(a));
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

constexpr int kUnroll = 4;
constexpr int kDropoutThreads = 256;
constexpr int kDropoutBlock = 8 * kDropoutThreads * kUnroll;  // elements of a block

// Eight elements of group g: limit = threshold << 16, so a word's high part
// passes when the word does, its low part when the word shifted up does.
template <typename Tx, typename Tr, bool RESIDUAL>
__device__ __forceinline__ void drop8(const Vec<Tx, 8>& x, const Vec<Tr, 8>& residual, int64_t g,
                                      uint64_t offset, uint2 key, uint32_t limit, float scale,
                                      float (&o)[8]) {
  const uint4 r = philox4x32_10(
      make_uint4(static_cast<uint32_t>(g), static_cast<uint32_t>(g >> 32),
                 static_cast<uint32_t>(offset), static_cast<uint32_t>(offset >> 32)),
      key);
  const uint32_t word[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    o[2 * j] = (word[j] << 16) >= limit ? to_f32(x.e[2 * j]) : 0.f;
    o[2 * j + 1] = word[j] >= limit ? to_f32(x.e[2 * j + 1]) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    o[j] = RESIDUAL ? fmaf(o[j], scale, to_f32(residual.e[j])) : o[j] * scale;
  }
}

// A thread takes kUnroll groups of eight elements, a block's width apart:
// the loads of all of them are in flight while their counters are hashed.
// VEC: x, residual and y are 16-byte aligned.
template <typename Tx, typename Tr, bool RESIDUAL, bool VEC>
__global__ void __launch_bounds__(kDropoutThreads)
    dropout_groups(const Tx* __restrict__ x, const Tr* __restrict__ residual, Tr* __restrict__ y,
                   int64_t count, uint32_t limit, float scale, uint64_t seed, uint64_t offset,
                   const int64_t* __restrict__ offset_dev) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  if (offset_dev != nullptr) offset = static_cast<uint64_t>(*offset_dev);
  const uint2 key = make_uint2(static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32));
  const int64_t start = static_cast<int64_t>(blockIdx.x) * kDropoutBlock;
  const int64_t first = start / 8 + threadIdx.x;
  x += start + threadIdx.x * 8;
  y += start + threadIdx.x * 8;
  if (RESIDUAL) residual += start + threadIdx.x * 8;
  Vec<Tx, 8> vx[kUnroll];
  Vec<Tr, 8> vr[kUnroll];
  if (VEC && start + kDropoutBlock <= count) {
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      vx[k] = load_vec<Tx, 8>(x + k * kDropoutThreads * 8);
      if (RESIDUAL) vr[k] = load_vec<Tr, 8>(residual + k * kDropoutThreads * 8);
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      float o[8];
      drop8<Tx, Tr, RESIDUAL>(vx[k], vr[k], first + k * kDropoutThreads, offset, key, limit, scale,
                              o);
      store_vec<Tr, 8>(y + k * kDropoutThreads * 8, o);
    }
    return;
  }
  // The last block, and views that no vector load fits.
  const int64_t left = count - start - threadIdx.x * 8;
#pragma unroll 1
  for (int k = 0; k < kUnroll; ++k) {
    const int at = k * kDropoutThreads * 8;
    if (at >= left) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = at + j < left;
      vx[0].e[j] = in ? x[at + j] : from_f32<Tx>(0.f);
      if (RESIDUAL) vr[0].e[j] = in ? residual[at + j] : from_f32<Tr>(0.f);
    }
    float o[8];
    drop8<Tx, Tr, RESIDUAL>(vx[0], vr[0], first + k * kDropoutThreads, offset, key, limit, scale, o);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (at + j < left) y[at + j] = from_f32<Tr>(o[j]);
    }
  }
}

template <typename Tx, typename Tr, bool RESIDUAL, bool VEC>
int launch_groups(const Dropout& a, cudaStream_t stream) {
  const uint32_t threshold = static_cast<uint32_t>(std::floor(a.p * 65536.0 + 0.5));
  if (threshold == 65536u) {
    // Everything is dropped: zeros, or the residual.
    const size_t bytes = static_cast<size_t>(a.count) * sizeof(Tr);
    if (!RESIDUAL) return launched(cudaMemsetAsync(a.y, 0, bytes, stream), "dropout");
    return launched(cudaMemcpyAsync(a.y, a.residual, bytes, cudaMemcpyDeviceToDevice, stream),
                    "dropout");
  }
  const float scale = static_cast<float>(65536.0 / (65536.0 - threshold));
  const int64_t blocks = (a.count + kDropoutBlock - 1) / kDropoutBlock;
  return launched(
      launch_kernel(dropout_groups<Tx, Tr, RESIDUAL, VEC>, dim3(static_cast<unsigned>(blocks)),
                    dim3(kDropoutThreads), 0, stream, 1, static_cast<const Tx*>(a.x),
                    static_cast<const Tr*>(a.residual), static_cast<Tr*>(a.y), a.count,
                    threshold << 16, scale, a.seed, a.offset, a.offset_dev),
      "dropout");
}

template <typename Tx, typename Tr>
int run_dropout(const Dropout& a, cudaStream_t stream) {
  const bool vec = vec_rows<Tx, 8>(a.x, 0, 8) && vec_rows<Tr, 8>(a.y, 0, 8) &&
                   vec_rows<Tr, 8>(a.residual, 0, 8);
  if (a.residual != nullptr) {
    return vec ? launch_groups<Tx, Tr, true, true>(a, stream)
               : launch_groups<Tx, Tr, true, false>(a, stream);
  }
  return vec ? launch_groups<Tx, Tr, false, true>(a, stream)
             : launch_groups<Tx, Tr, false, false>(a, stream);
}

}  // namespace

int launch_dropout(const Dropout& a, cudaStream_t stream) {
  if (a.x_dtype == CCV_DTYPE_BF16) {
    return a.y_dtype == CCV_DTYPE_F32 ? run_dropout<__nv_bfloat16, float>(a, stream)
                                      : run_dropout<__nv_bfloat16, __nv_bfloat16>(a, stream);
  }
  if (a.x_dtype == CCV_DTYPE_F16) {
    return a.y_dtype == CCV_DTYPE_F32 ? run_dropout<__half, float>(a, stream)
                                      : run_dropout<__half, __half>(a, stream);
  }
  if (a.y_dtype == CCV_DTYPE_BF16) return run_dropout<float, __nv_bfloat16>(a, stream);
  if (a.y_dtype == CCV_DTYPE_F16) return run_dropout<float, __half>(a, stream);
  return run_dropout<float, float>(a, stream);
}

}  // namespace ccv
