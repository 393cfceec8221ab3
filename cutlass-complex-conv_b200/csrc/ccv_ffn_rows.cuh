// Gated feed-forward block for a few rows (one token to a small batch): the
// time is that of reading the three weights once, so they are streamed from
// global memory straight into the registers that feed mma.sync, 16 bytes a
// lane, with no shared-memory stage and no tile of 128 rows to pad.  (The
// tcgen05 kernel reads operands from shared memory in tiles of 256 rows; with
// few rows its multiplications are free but its grid is too small to keep
// enough loads in flight.)
//
// A warp multiplies 16 weight rows by up to 8 NT tokens over its share of the
// reduction: m16n8k16 with the weights as the 16-row operand.  The product
// sums over k in any order, so both operands take a permuted k: lane t of a
// quad loads 8 adjacent k (16 bytes) and feeds k 0-3 to one instruction and
// 4-7 to the next.  The gate kernel's 16 rows are 8 gate rows and the 8 up
// rows of the same outputs: g and u of one output meet in one lane.
//
// The reduction is shared by the warps of a block, and for the down
// projection by the blocks of a cluster; partial sums are added in a fixed
// order.  The down kernel loads its first weights before it waits for the
// gate kernel (they do not depend on it), so the two streams of weights run
// into each other.
//
// Measured on B200: one row at 1024 x 4096 bf16 8.7-9.9 us (25 MB of weights,
// 2.5-2.9 TB/s: two dependent launches of about 4 us), at 2048 x 8192 20.5 us
// (4.9 TB/s); 16 rows 13.4 and 32 us.
#pragma once

#include "ccv_ffn_gemm.cuh"
#include "ccv_internal.h"
#include "ccv_ptx.cuh"
#include "ccv_tokens.cuh"

namespace ccv {
namespace ffn {

constexpr int kRowsWarps = 8;
constexpr int kRowsThreads = 32 * kRowsWarps;
constexpr int kChunk = 32;   // k per lane quad and load: 4 lanes x 8
constexpr int kBatch = 4;    // chunks loaded together

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Elements k .. k + 7 of a row of `n`, zero past its end; the row is null
// outside the matrix.  VEC: rows are 16-byte aligned and n % 8 == 0.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int k, int n) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (row == nullptr || k >= n) return v;
  if (VEC) return *reinterpret_cast<const uint4*>(row + k);
  uint16_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = k + i < n ? row[k + i] : static_cast<uint16_t>(0);
  v.x = e[0] | static_cast<uint32_t>(e[1]) << 16;
  v.y = e[2] | static_cast<uint32_t>(e[3]) << 16;
  v.z = e[4] | static_cast<uint32_t>(e[5]) << 16;
  v.w = e[6] | static_cast<uint32_t>(e[7]) << 16;
  return v;
}

// acc += the two weight rows' (low: rows 0-7 of the instruction, high: rows
// 8-15) products with NT groups of 8 tokens over k0 <= k < k1.  `first`:
// weights of the first batch, loaded by the caller.
template <typename T, int NT, bool VEC_W, bool VEC_X>
struct Stream {
  uint4 lo[kBatch], hi[kBatch];

  __device__ __forceinline__ void load(const uint16_t* low, const uint16_t* high, int k, int k1,
                                       int n) {
#pragma unroll
    for (int c = 0; c < kBatch; ++c) {
      const int kk = k + c * kChunk;
      lo[c] = load8<VEC_W>(kk < k1 ? low : nullptr, kk, n);
      hi[c] = load8<VEC_W>(kk < k1 ? high : nullptr, kk, n);
    }
  }
  // For two groups of tokens their values are loaded ahead of the first
  // multiplication (16 rows at 1024 x 4096: 14.7 -> 13.4 us); for one, the
  // registers that takes cost more warps than it gains (8.7 -> 10.4 us).
  __device__ __forceinline__ void multiply(float (&acc)[NT][4], const uint16_t* const (&tok)[NT],
                                           int k, int k1, int n) {
    constexpr bool kAhead = NT > 1;
    uint4 x[kAhead ? kBatch : 1][NT];
    auto load = [&](int c, uint4 (&v)[NT]) {
      const int kk = k + c * kChunk;
#pragma unroll
      for (int t = 0; t < NT; ++t) v[t] = load8<VEC_X>(kk < k1 ? tok[t] : nullptr, kk, n);
    };
    if constexpr (kAhead) {
#pragma unroll
      for (int c = 0; c < kBatch; ++c) load(c, x[c]);
    }
#pragma unroll
    for (int c = 0; c < kBatch; ++c) {
      const int kk = k + c * kChunk;
      if (kk - (kk & 31) < k1) {  // the whole quad: k is the lane's, its chunk the warp's
        if constexpr (!kAhead) load(c, x[0]);
        const uint4 (&v)[NT] = x[kAhead ? c : 0];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma_16816(acc[t], lo[c].x, hi[c].x, lo[c].y, hi[c].y, v[t].x, v[t].y, T());
          mma_16816(acc[t], lo[c].z, hi[c].z, lo[c].w, hi[c].w, v[t].z, v[t].w, T());
        }
      }
    }
  }
};

struct RowsParams {
  const uint16_t* x;       // [rows][k]: tokens (gate) or h (down)
  int64_t x_stride;
  const uint16_t *w0, *w1; // gate and up [out][k]; down [out][k] and null
  uint16_t *out, *g, *u, *next;  // h and the planes of g and u (null without saving); y
  int64_t out_stride;
  int rows, k, outputs;
  int blocks_per_cta;      // gate: groups of 8 outputs per block
  int act;
};

// h (and g, u) for 8 outputs per group; columns past the last output up to
// the next multiple of 8 are written as zeros (the down kernel reads whole
// groups of 8).
template <typename T, int NT, bool VEC>
__global__ void __launch_bounds__(kRowsThreads)
    ffn_rows_gate(const RowsParams p) {
  __shared__ float part[kRowsWarps][16][8 * NT + 1];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane >> 2, t4 = lane & 3;
  const uint16_t* tok[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int m = t * 8 + quad;
    tok[t] = m < p.rows ? p.x + m * p.x_stride : nullptr;
  }
  // Each warp's share of the reduction: whole chunks, so that no lane of a
  // quad leaves its instruction.
  const int chunks = (p.k + kChunk - 1) / kChunk;
  const int c0 = chunks * warp / kRowsWarps, c1 = chunks * (warp + 1) / kRowsWarps;
  for (int b = 0; b < p.blocks_per_cta; ++b) {
    const int o0 = (blockIdx.x * p.blocks_per_cta + b) * 8;
    if (o0 >= p.outputs) break;
    const int o = o0 + quad;
    const uint16_t* low = o < p.outputs ? p.w0 + static_cast<int64_t>(o) * p.k : nullptr;
    const uint16_t* high = o < p.outputs ? p.w1 + static_cast<int64_t>(o) * p.k : nullptr;
    float acc[NT][4] = {};
    Stream<T, NT, VEC, VEC> s;
    for (int c = c0; c < c1; c += kBatch) {
      s.load(low, high, c * kChunk + t4 * 8, c1 * kChunk, p.k);
      s.multiply(acc, tok, c * kChunk + t4 * 8, c1 * kChunk, p.k);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      part[warp][quad][t * 8 + 2 * t4] = acc[t][0];
      part[warp][quad][t * 8 + 2 * t4 + 1] = acc[t][1];
      part[warp][quad + 8][t * 8 + 2 * t4] = acc[t][2];
      part[warp][quad + 8][t * 8 + 2 * t4 + 1] = acc[t][3];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 8 * 8 * NT; e += kRowsThreads) {
      const int m = e >> 3, f = e & 7;
      if (m < p.rows) {
        float g = 0.f, u = 0.f;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {
          g += part[w][f][m];
          u += part[w][f + 8][m];
        }
        float value, slope;
        if (p.act == CCV_ACTIVATION_SILU) {
          activation<CCV_ACTIVATION_SILU>(g, value, slope);
        } else {
          activation<CCV_ACTIVATION_GELU>(g, value, slope);
        }
        const int64_t at = m * p.out_stride + o0 + f;
        // Outputs past the last one have g = u = 0 and write the zero padding.
        reinterpret_cast<T*>(p.out)[at] = from_f32<T>(value * u);
        if (p.g != nullptr) {
          const uint32_t gb = __float_as_uint(g), ub = __float_as_uint(u);
          p.g[at] = static_cast<uint16_t>(gb >> 16);
          p.u[at] = static_cast<uint16_t>(ub >> 16);
          p.next[at] = static_cast<uint16_t>(next_bytes(gb, ub, gb, ub));
        }
      }
    }
    __syncthreads();
  }
}

// y for 16 outputs per cluster; the cluster's blocks and their warps share
// the reduction.
template <typename T, int NT, bool VEC_W>
__global__ void __launch_bounds__(kRowsThreads)
    ffn_rows_down(const RowsParams p) {
  __shared__ float part[kRowsWarps][16][8 * NT + 1];
  __shared__ __align__(16) float sum[16 * 8 * NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane >> 2, t4 = lane & 3;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int size = static_cast<int>(ptx::cluster_nctarank());
  const int o0 = (blockIdx.x / size) * 16;
  const uint16_t* low = o0 + quad < p.outputs ? p.w0 + static_cast<int64_t>(o0 + quad) * p.k : nullptr;
  const uint16_t* high =
      o0 + quad + 8 < p.outputs ? p.w0 + static_cast<int64_t>(o0 + quad + 8) * p.k : nullptr;
  const int chunks = (p.k + kChunk - 1) / kChunk;
  const int share = rank * kRowsWarps + warp, shares = size * kRowsWarps;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * share / shares);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (share + 1) / shares);
  Stream<T, NT, VEC_W, true> s;
  // The weights are inputs of the whole call, complete before the gate kernel
  // began; only h is its result.
  s.load(low, high, c0 * kChunk + t4 * 8, c1 * kChunk, p.k);
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const uint16_t* tok[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int m = t * 8 + quad;
    tok[t] = m < p.rows ? p.x + m * p.x_stride : nullptr;
  }
  float acc[NT][4] = {};
  for (int c = c0; c < c1; c += kBatch) {
    if (c != c0) s.load(low, high, c * kChunk + t4 * 8, c1 * kChunk, p.k);
    s.multiply(acc, tok, c * kChunk + t4 * 8, c1 * kChunk, p.k);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    part[warp][quad][t * 8 + 2 * t4] = acc[t][0];
    part[warp][quad][t * 8 + 2 * t4 + 1] = acc[t][1];
    part[warp][quad + 8][t * 8 + 2 * t4] = acc[t][2];
    part[warp][quad + 8][t * 8 + 2 * t4 + 1] = acc[t][3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * 8 * NT; e += kRowsThreads) {
    const int m = e >> 4, o = e & 15;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) v += part[w][o][m];
    sum[e] = v;
  }
  ptx::cluster_sync();
  if (rank == 0) {
    for (int e = threadIdx.x; e < 16 * 8 * NT / 4; e += kRowsThreads) {
      const int m = e >> 2, o = (e & 3) * 4;
      if (m < p.rows) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < size; ++r) {
          const float4 q = ptx::ld_shared_cluster_v4_ordered(ptx::mapa_shared(ptx::smem_u32(sum + 4 * e), r));
          v.x += q.x;
          v.y += q.y;
          v.z += q.z;
          v.w += q.w;
        }
        const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (o0 + o + j < p.outputs) {
            reinterpret_cast<T*>(p.out)[m * p.out_stride + o0 + o + j] = from_f32<T>(f[j]);
          }
        }
      }
    }
  }
  ptx::cluster_sync();  // the other blocks' sums stay until rank 0 has read them
}

}  // namespace ffn
}  // namespace ccv
