// Layer norm over rows of features, forward and backward.
//
//   mean = sum_j x_j / D,  var = sum_j (x_j - mean)^2 / D,  r = 1/sqrt(var + eps)
//   y_j = (x_j - mean) r w_j + b_j
// and with z_j = (x_j - mean) r, t_j = dy_j w_j:
//   dx_j = r (t_j - sum t / D - z_j sum(t z) / D)
//   dw_j = sum_rows dy_j z_j,   db_j = sum_rows dy_j
//
// Both directions are bound by memory: the forward pass reads x and writes y
// once, the backward pass reads x and dy and writes dx once.  One block of up
// to 512 threads per SM walks the rows; a group of G threads holds a row, 16
// elements each (G a power of two within a warp, then whole warps: narrow
// rows share a warp and cost few shuffles per element).  Every thread copies
// the vectors it will use itself into a shared-memory ring some rows ahead
// (cp.async), so 64 KB and more per SM are in flight at all times and no
// barrier guards the ring.  Its columns stay the same from row to row: the
// weights are in registers, and the backward pass sums dw and db over the
// rows there, reading nothing twice; blocks leave fp32 partial sums that a
// second launch adds in block order (deterministic).  Measured on B200, 200704
// x 256, fp32 x, bf16 y: forward 49.9 us (6.2 TB/s, 96 % of the copy rate),
// backward 86-90 us (5.7-6.0 TB/s); bf16 12545 x 1024 13.6 and 22 us.
//
// Rows that 16-byte vectors do not divide go in pairs of elements where those
// divide them.  Dense rows of odd width start at any element of a vector: a
// group's rows are then a multiple of V rows apart, so they all start at the
// same one, and the group's vectors are shifted by it; the first and the last
// may hold elements of the row's neighbours, which a bit mask excludes
// (SHIFT).  Other layouts, and rows shorter than the vectors would reach past
// them, take single elements, and rows wider than 8192 the kernels further
// down.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "ccv_internal.h"
#include "ccv_norm_shift.h"
#include "ccv_ptx.cuh"
#include "ccv_tokens.cuh"

namespace ccv {

namespace {

constexpr int kHeld = 16;        // elements of a row per thread
constexpr int kThreads = 512;    // most threads of a block
constexpr int kRingBytes = 196 * 1024;

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES)
                 : "memory");
  }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Sums over the G threads of a group: shuffles within a warp, then (G > 32)
// an exchange through shared memory, added in warp order.  Successive calls
// alternate between the halves of `red` [2][warps of the block][N].
template <int N>
struct GroupSum {
  int g, group;
  float* red;
  int parity = 0;

  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (o < g) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      }
    }
    if (g <= 32) return;
    float* mine = red + parity * (kThreads / 32) * N;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) mine[(threadIdx.x >> 5) * N + i] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(g) : "memory");
    const int warps = g >> 5;
    const float* first = mine + group * warps * N;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    for (int w = 0; w < warps; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += first[w * N + i];
    }
    parity ^= 1;
  }
};

// A thread's vectors of one tensor in one ring stage: 16 elements in VPT
// vectors of V, each in pieces of up to 16 bytes.
template <typename T, int V>
struct Held {
  static constexpr int kVpt = kHeld / V;
  static constexpr int kPiece = V * sizeof(T) < 16 ? V * sizeof(T) : 16;
  static constexpr int kPieces = V * sizeof(T) / kPiece;
  static constexpr int kBytes = kHeld * sizeof(T);  // per thread
  static __device__ __forceinline__ uint32_t address(uint32_t stage, int i, int q) {
    return stage + ((i * kPieces + q) * blockDim.x + threadIdx.x) * kPiece;
  }
  static __device__ __forceinline__ void zero(uint32_t stage, int i) {
#pragma unroll
    for (int q = 0; q < kPieces; ++q) {
      const uint32_t at = address(stage, i, q);
      if constexpr (kPiece == 16) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
      } else if constexpr (kPiece == 8) {
        asm volatile("st.shared.v2.b32 [%0], {%1, %1};" ::"r"(at), "r"(0) : "memory");
      } else if constexpr (kPiece == 4) {
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(0) : "memory");
      }
    }
  }
  // Vector i from column c of `row` on.
  static __device__ __forceinline__ void fetch(uint32_t stage, int i, const T* row, int c) {
#pragma unroll
    for (int q = 0; q < kPieces; ++q) {
      copy_async<kPiece>(address(stage, i, q), reinterpret_cast<const char*>(row + c) + q * kPiece);
    }
  }
  // The same for a vector that reaches past the tensor's end.
  static __device__ __forceinline__ void fetch_end(uint32_t stage, int i, const T* row, int c,
                                                   int features) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (c + j < features) {
        const uint32_t to =
            address(stage, i, j * sizeof(T) / kPiece) + (j * sizeof(T)) % kPiece;
        if constexpr (sizeof(T) == 4) {
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(to),
                       "r"(*reinterpret_cast<const uint32_t*>(row + c + j))
                       : "memory");
        } else {
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(to),
                       "h"(*reinterpret_cast<const uint16_t*>(row + c + j))
                       : "memory");
        }
      }
    }
  }
  static __device__ __forceinline__ Vec<T, V> read(const uint8_t* stage, int i) {
    Vec<T, V> v;
    using Piece = std::conditional_t<kPiece == 16, uint4, std::conditional_t<kPiece == 8, uint2,
                  std::conditional_t<kPiece == 4, uint32_t, uint16_t>>>;
#pragma unroll
    for (int q = 0; q < kPieces; ++q) {
      reinterpret_cast<Piece*>(&v)[q] = *reinterpret_cast<const Piece*>(
          stage + ((i * kPieces + q) * blockDim.x + threadIdx.x) * kPiece);
    }
    return v;
  }
};

// Zeroes the elements of a vector at column c that lie outside the row.
template <typename T, int V>
__device__ __forceinline__ void clip(Vec<T, V>& v, int c, int features) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (c + j < 0 || c + j >= features) v.e[j] = from_f32<T>(0.f);
  }
}

// Bits of the elements of a thread's vectors that lie in the row (shifted
// vectors: the first may begin in the row before, the last end in the next).
template <int V>
struct Inside {
  uint32_t bits = 0;
  __device__ __forceinline__ void add(int i, int c, int features) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (c + j >= 0 && c + j < features) bits |= 1u << (i * V + j);
    }
  }
  __device__ __forceinline__ bool element(int i, int j) const {
    return (bits >> (i * V + j) & 1u) != 0;
  }
  __device__ __forceinline__ bool whole(int i) const {
    constexpr uint32_t all = (1u << V) - 1u;
    return (bits >> (i * V) & all) == all;
  }
};

// Ring stages for `bytes` per thread and row.
template <int BYTES>
constexpr int kRingStages =
    kRingBytes / (kThreads * BYTES) < 6 ? kRingBytes / (kThreads * BYTES) : 6;

// Forward, rows of up to 8192 features.
template <typename Tx, typename Tw, typename Ty, int V, bool SHIFT>
__global__ void __launch_bounds__(kThreads, 1)
    norm_forward_ring(const Tx* __restrict__ x, int64_t x_stride, const Tw* __restrict__ w,
                      const Tw* __restrict__ b, float eps, Ty* __restrict__ y,
                      float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows,
                      int features, int g) {
  using Hx = Held<Tx, V>;
  constexpr int VPT = Hx::kVpt;
  constexpr int S = kRingStages<Hx::kBytes>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[2 * (kThreads / 32) * 2];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int group = threadIdx.x / g;
  const int lane = threadIdx.x - group * g;
  const int per_block = blockDim.x / g;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per_block;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
  const int shift = SHIFT ? shift_of_row(first + group, features, V) : 0;
  auto column = [&](int i) { return shifted_column(i, g, lane, V, shift); };
  Inside<V> inside;
  if (SHIFT) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) inside.add(i, column(i), features);
  }
  const uint32_t ring_base = ptx::smem_u32(ring);
  const uint32_t stage_bytes = blockDim.x * Hx::kBytes;
  auto fetch = [&](int stage, int64_t r) {
    if (r < rows) {
      const Tx* row = x + r * x_stride;
      const uint32_t at = ring_base + stage * stage_bytes;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = column(i);
        if (SHIFT && past_the_end(r, rows, c, features, V)) {
          Hx::fetch_end(at, i, row, c, features);
        } else if (c < features) {
          Hx::fetch(at, i, row, c);
        }
      }
    }
    copy_commit();
  };
  // Vectors past the row's end stay zero.
  for (int k = 0; k < S; ++k) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (column(i) + V > features) Hx::zero(ring_base + k * stage_bytes, i);
    }
    fetch(k, first + group + k * step);
  }
  float wt[VPT][V], bs[VPT][V];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = column(i);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool in = c + j >= 0 && c + j < features;
      wt[i][j] = in && w != nullptr ? to_f32(w[c + j]) : 1.f;
      bs[i][j] = in && b != nullptr ? to_f32(b[c + j]) : 0.f;
    }
  }
  GroupSum<2> total{g, group, red};
  const float n = static_cast<float>(features), inv = 1.f / n;
  int stage = 0;
  // Two rows at a time: one exchange serves both sums, and the rows' chains of
  // dependent operations overlap.  The block's groups walk together: every
  // thread takes part in each sum.
  for (int64_t r0 = first; r0 < rows; r0 += 2 * step) {
    copy_wait<S - 2>();
    float v[2][VPT][V];
    float sum[2] = {0.f, 0.f}, mean[2], sq[2] = {0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const Vec<Tx, V> q = Hx::read(ring + stage * stage_bytes, i);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[h][i][j] = !SHIFT || inside.element(i, j) ? to_f32(q.e[j]) : 0.f;
          sum[h] += v[h][i][j];
        }
      }
      fetch(stage, r0 + group + (S + h) * step);
      stage = stage + 1 == S ? 0 : stage + 1;
    }
    total(sum);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mean[h] = sum[h] / n;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = column(i);
#pragma unroll
        for (int j = 0; j < V; ++j) v[h][i][j] -= mean[h];
        if (SHIFT) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if (inside.element(i, j)) sq[h] = fmaf(v[h][i][j], v[h][i][j], sq[h]);
          }
        } else if (c < features) {
#pragma unroll
          for (int j = 0; j < V; ++j) sq[h] = fmaf(v[h][i][j], v[h][i][j], sq[h]);
        }
      }
    }
    total(sq);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t r = r0 + group + h * step;
      if (r >= rows) break;
      const float rstd = rsqrtf(sq[h] * inv + eps);
      Ty* yr = y + r * features;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = column(i);
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = fmaf(v[h][i][j] * rstd, wt[i][j], bs[i][j]);
        if (SHIFT ? inside.whole(i) : c < features) {
          store_vec<Ty, V>(yr + c, o);
        } else if (SHIFT) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if (inside.element(i, j)) yr[c + j] = from_f32<Ty>(o[j]);
          }
        }
      }
      if (lane == 0) {
        if (mean_out != nullptr) mean_out[r] = mean[h];
        if (rstd_out != nullptr) rstd_out[r] = rstd;
      }
    }
  }
}

// Backward, rows of up to 8192 features; partial: [blocks][2][features].
// V = 1: single elements straight from global memory.
template <typename Tx, typename Tw, typename Ty, int V, bool SHIFT>
__global__ void __launch_bounds__(kThreads, 1)
    norm_backward_ring(const Ty* __restrict__ dy, int64_t dy_stride, const Tx* __restrict__ x,
                       int64_t x_stride, const float* __restrict__ mean_in,
                       const float* __restrict__ rstd_in, const Tw* __restrict__ w,
                       Tx* __restrict__ dx, float* __restrict__ partial, int64_t rows,
                       int features, int g) {
  using Hx = Held<Tx, V>;
  using Hy = Held<Ty, V>;
  constexpr int VPT = Hx::kVpt;
  constexpr int S = kRingStages<Hx::kBytes + Hy::kBytes>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[2 * (kThreads / 32) * 2];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int group = threadIdx.x / g;
  const int lane = threadIdx.x - group * g;
  const int per_block = blockDim.x / g;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per_block;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
  const int shift = SHIFT ? shift_of_row(first + group, features, V) : 0;
  auto column = [&](int i) { return shifted_column(i, g, lane, V, shift); };
  const uint32_t ring_base = ptx::smem_u32(ring);
  const uint32_t x_bytes = blockDim.x * Hx::kBytes;
  const uint32_t stage_bytes = x_bytes + blockDim.x * Hy::kBytes;
  auto fetch = [&](int stage, int64_t r) {
    if constexpr (V > 1) {
      const uint32_t at = ring_base + stage * stage_bytes;
      if (r < rows) {
        const Tx* xr = x + r * x_stride;
        const Ty* gr = dy + r * dy_stride;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int c = column(i);
          if (SHIFT && past_the_end(r, rows, c, features, V)) {
            Hx::fetch_end(at, i, xr, c, features);
            Hy::fetch_end(at + x_bytes, i, gr, c, features);
          } else if (c < features) {
            Hx::fetch(at, i, xr, c);
            Hy::fetch(at + x_bytes, i, gr, c);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) Hy::zero(at + x_bytes, i);
      }
      copy_commit();
    }
  };
  // Vectors past the row's end stay zero in dy, and rows past the last one
  // become zero: they add nothing to any sum.  (x must only be finite there.)
  if constexpr (V > 1) {
    for (int k = 0; k < S; ++k) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (column(i) + V > features || first + group + k * step >= rows) {
          Hx::zero(ring_base + k * stage_bytes, i);
          Hy::zero(ring_base + k * stage_bytes + x_bytes, i);
        }
      }
      fetch(k, first + group + k * step);
    }
  }
  const float inv = 1.f / static_cast<float>(features);
  float wt[VPT][V], dw[VPT][V] = {}, db[VPT][V] = {};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = column(i);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      wt[i][j] = w != nullptr && c + j >= 0 && c + j < features ? to_f32(w[c + j]) : 1.f;
    }
  }
  float mean = 0.f, rstd = 0.f;
  if (first + group < rows) {
    mean = mean_in[first + group];
    rstd = rstd_in[first + group];
  }
  GroupSum<2> total{g, group, red};
  int stage = 0;
  // The block's groups walk together: every thread takes part in each sum.
  for (int64_t r0 = first; r0 < rows; r0 += step) {
    const int64_t r = r0 + group;
    const bool live = r < rows;
    const float scale = rstd;
    if constexpr (V > 1) copy_wait<S - 1>();
    float z[VPT][V], t[VPT][V];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = column(i);
      Vec<Tx, V> qx;
      Vec<Ty, V> qg;
      if constexpr (V > 1) {
        qx = Hx::read(ring + stage * stage_bytes, i);
        qg = Hy::read(ring + stage * stage_bytes + x_bytes, i);
        // (A bit mask as in the forward kernel does not fit in the registers:
        // 12545 x 1001 fp32 43 us against 36.)
        if (SHIFT && (c < 0 || c + V > features)) {
          clip(qx, c, features);
          clip(qg, c, features);
        }
      } else {
        qx.e[0] = from_f32<Tx>(0.f);
        qg.e[0] = from_f32<Ty>(0.f);
        if (live && c < features) {
          qx.e[0] = x[r * x_stride + c];
          qg.e[0] = dy[r * dy_stride + c];
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = to_f32(qg.e[j]);
        z[i][j] = (to_f32(qx.e[j]) - mean) * scale;
        t[i][j] = d * wt[i][j];
        dw[i][j] = fmaf(d, z[i][j], dw[i][j]);
        db[i][j] += d;
        sum[0] += t[i][j];
        sum[1] = fmaf(t[i][j], z[i][j], sum[1]);
      }
    }
    fetch(stage, r + S * step);
    stage = stage + 1 == S ? 0 : stage + 1;
    if (r + step < rows) {
      mean = mean_in[r + step];
      rstd = rstd_in[r + step];
    }
    total(sum);
    if (!live || dx == nullptr) continue;
    const float a = sum[0] * inv, c1 = sum[1] * inv;
    Tx* out = dx + r * features;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = column(i);
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = scale * (t[i][j] - a - z[i][j] * c1);
      if (!SHIFT || (c >= 0 && c + V <= features)) {
        if (c < features) store_vec<Tx, V>(out + c, o);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (c + j >= 0 && c + j < features) out[c + j] = from_f32<Tx>(o[j]);
        }
      }
    }
  }
  // The groups' sums side by side in the ring's memory, then added in order.
  copy_wait<0>();
  __syncthreads();
  float* sums = reinterpret_cast<float*>(ring);  // [groups][2][features]
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = column(i);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (c + j >= 0 && c + j < features) {
        sums[(group * 2) * features + c + j] = dw[i][j];
        sums[(group * 2 + 1) * features + c + j] = db[i][j];
      }
    }
  }
  __syncthreads();
  float* out = partial + static_cast<int64_t>(blockIdx.x) * 2 * features;
  for (int c = threadIdx.x; c < 2 * features; c += blockDim.x) {
    float v = 0.f;
    for (int k = 0; k < per_block; ++k) v += sums[k * 2 * features + c];
    out[c] = v;
  }
}

// Sum over a row's G threads where the group is the block for G > 32.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int g, float (*red)[N]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (o < g) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
  }
  if (g > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[warp][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    const int warps = g >> 5;
    for (int w = 0; w < warps; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += red[w][i];
    }
  }
}

// Forward without the ring, VPT vectors of V elements per thread, one row per
// group and launch: rows of more than 8192 features, and single elements.
template <typename Tx, typename Tw, typename Ty, int V, int VPT>
__global__ void __launch_bounds__(1024, 1)
    norm_forward_held(const Tx* __restrict__ x, int64_t x_stride, const Tw* __restrict__ w,
                      const Tw* __restrict__ b, float eps, Ty* __restrict__ y,
                      float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows,
                      int features, int g) {
  __shared__ float red[2][32][1];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int lane = threadIdx.x & (g > 32 ? ~0 : g - 1);
  const int per_block = g > 32 ? 1 : blockDim.x / g;
  const int64_t row =
      static_cast<int64_t>(blockIdx.x) * per_block + (g > 32 ? 0 : threadIdx.x / g);
  const bool live = row < rows;
  const Tx* xr = x + (live ? row : 0) * x_stride;
  Vec<Tx, V> raw[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (i * g + lane) * V;
    if (c < features) raw[i] = load_vec<Tx, V>(xr + c);
  }
  float sum[1] = {0.f};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if ((i * g + lane) * V < features) {
#pragma unroll
      for (int j = 0; j < V; ++j) sum[0] += to_f32(raw[i].e[j]);
    }
  }
  group_sum<1>(sum, g, red[0]);
  const float mean = sum[0] / static_cast<float>(features);
  float sq[1] = {0.f};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if ((i * g + lane) * V < features) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = to_f32(raw[i].e[j]) - mean;
        sq[0] = fmaf(d, d, sq[0]);
      }
    }
  }
  group_sum<1>(sq, g, red[1]);
  const float rstd = rsqrtf(sq[0] / static_cast<float>(features) + eps);
  if (!live) return;
  Ty* yr = y + row * features;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (i * g + lane) * V;
    if (c < features) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = (to_f32(raw[i].e[j]) - mean) * rstd;
      if (w != nullptr) {
        const Vec<Tw, V> wv = load_vec<Tw, V>(w + c);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] *= to_f32(wv.e[j]);
      }
      if (b != nullptr) {
        const Vec<Tw, V> bv = load_vec<Tw, V>(b + c);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] += to_f32(bv.e[j]);
      }
      store_vec<Ty, V>(yr + c, o);
    }
  }
  if (lane == 0) {
    if (mean_out != nullptr) mean_out[row] = mean;
    if (rstd_out != nullptr) rstd_out[row] = rstd;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp per row; the row is read three times (from L1/L2 after the first).
// For rows of more than 32768 features.
template <typename Tx, typename Tw, typename Ty>
__global__ void norm_forward_rows(const Tx* __restrict__ x, int64_t x_stride,
                                  const Tw* __restrict__ w, const Tw* __restrict__ b, float eps,
                                  Ty* __restrict__ y, float* __restrict__ mean_out,
                                  float* __restrict__ rstd_out, int64_t rows, int64_t features) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
       row < rows; row += warps) {
    const Tx* xr = x + row * x_stride;
    float s = 0.f;
    for (int64_t j = lane; j < features; j += 32) s += to_f32(xr[j]);
    const float mean = warp_sum(s) / static_cast<float>(features);
    float q = 0.f;
    for (int64_t j = lane; j < features; j += 32) {
      const float d = to_f32(xr[j]) - mean;
      q += d * d;
    }
    const float rstd = rsqrtf(warp_sum(q) / static_cast<float>(features) + eps);
    for (int64_t j = lane; j < features; j += 32) {
      float v = (to_f32(xr[j]) - mean) * rstd;
      if (w != nullptr) v *= to_f32(w[j]);
      if (b != nullptr) v += to_f32(b[j]);
      y[row * features + j] = from_f32<Ty>(v);
    }
    if (lane == 0) {
      if (mean_out != nullptr) mean_out[row] = mean;
      if (rstd_out != nullptr) rstd_out[row] = rstd;
    }
  }
}

// dx of rows wider than a block's registers hold, one warp per row.
template <typename Tx, typename Tw, typename Ty>
__global__ void norm_backward_rows(const Ty* __restrict__ dy, int64_t dy_stride,
                                   const Tx* __restrict__ x, int64_t x_stride,
                                   const float* __restrict__ mean_in,
                                   const float* __restrict__ rstd_in, const Tw* __restrict__ w,
                                   Tx* __restrict__ dx, int64_t rows, int64_t features) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  const float inv = 1.f / static_cast<float>(features);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
       row < rows; row += warps) {
    const float mean = mean_in[row], rstd = rstd_in[row];
    float st = 0.f, stz = 0.f;
    for (int64_t j = lane; j < features; j += 32) {
      const float t = to_f32(dy[row * dy_stride + j]) * (w != nullptr ? to_f32(w[j]) : 1.f);
      st += t;
      stz += t * ((to_f32(x[row * x_stride + j]) - mean) * rstd);
    }
    st = warp_sum(st) * inv;
    stz = warp_sum(stz) * inv;
    for (int64_t j = lane; j < features; j += 32) {
      const float t = to_f32(dy[row * dy_stride + j]) * (w != nullptr ? to_f32(w[j]) : 1.f);
      const float z = (to_f32(x[row * x_stride + j]) - mean) * rstd;
      dx[row * features + j] = from_f32<Tx>(rstd * (t - st - z * stz));
    }
  }
}

constexpr int kColThreadsX = 32, kColThreadsY = 8;

// Their column sums, over one slice of rows: partial [slices][2][features].
template <typename Tx, typename Ty>
__global__ void norm_backward_columns(const Ty* __restrict__ dy, int64_t dy_stride,
                                      const Tx* __restrict__ x, int64_t x_stride,
                                      const float* __restrict__ mean_in,
                                      const float* __restrict__ rstd_in,
                                      float* __restrict__ partial, int64_t rows, int64_t features) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  __shared__ float sh[2][kColThreadsY][kColThreadsX];
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kColThreadsX + threadIdx.x;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
  float dw = 0.f, db = 0.f;
  if (j < features) {
    for (int64_t r = r0 + threadIdx.y; r < r1; r += kColThreadsY) {
      const float g = to_f32(dy[r * dy_stride + j]);
      dw += g * ((to_f32(x[r * x_stride + j]) - mean_in[r]) * rstd_in[r]);
      db += g;
    }
  }
  sh[0][threadIdx.y][threadIdx.x] = dw;
  sh[1][threadIdx.y][threadIdx.x] = db;
  __syncthreads();
  if (threadIdx.y < 2 && j < features) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kColThreadsY; ++i) s += sh[threadIdx.y][i][threadIdx.x];
    partial[(static_cast<int64_t>(blockIdx.y) * 2 + threadIdx.y) * features + j] = s;
  }
}

// dweight and dbias from the blocks' partial sums [slices][2][features]: 32
// columns per block, each warp takes every 32nd slice (its few loads are in
// flight together), then they add up in warp order.
template <typename Tw>
__global__ void __launch_bounds__(1024) norm_backward_reduce(const float* __restrict__ partial,
                                                             int slices, Tw* __restrict__ dw,
                                                             Tw* __restrict__ db,
                                                             int64_t features) {
  __shared__ float sh[2][32][33];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sw = 0.f, sb = 0.f;
  if (j < features) {
#pragma unroll 8
    for (int s = warp; s < slices; s += 32) {
      sw += partial[(static_cast<int64_t>(s) * 2) * features + j];
      sb += partial[(static_cast<int64_t>(s) * 2 + 1) * features + j];
    }
  }
  sh[0][warp][lane] = sw;
  sh[1][warp][lane] = sb;
  __syncthreads();
  // Warp w adds columns' warps: lane l of warp w holds warp l's sum of column w.
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + warp;
  if (col >= features) return;
  float a = sh[0][lane][warp], b = sh[1][lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (lane == 0) {
    if (dw != nullptr) dw[col] = from_f32<Tw>(a);
    if (db != nullptr) db[col] = from_f32<Tw>(b);
  }
}

int column_slices(int64_t rows) {
  const int64_t s = (rows + 63) / 64;
  return static_cast<int>(s < 1 ? 1 : (s > 128 ? 128 : s));
}

}  // namespace

namespace {

// Threads per row for `per` elements each: a power of two within a warp,
// whole warps above; 0 when more than `most` would be needed.
int group_size(int64_t features, int per, int most) {
  const int64_t need = (features + per - 1) / per;
  if (need > most) return 0;
  if (need > 32) return static_cast<int>((need + 31) / 32 * 32);
  int g = 1;
  while (g < need) g *= 2;
  return g;
}

// Grid of the ring kernels.
struct Rings {
  int g, per_block, blocks;
};

// Groups of g threads; v > 1: a group's rows start at the same element of a
// vector of v, so they are a multiple of v rows apart.
Rings plan_rings(int64_t rows, int g, int v) {
  const int sms = device_sm_count();
  Rings p;
  p.g = g;
  p.per_block = static_cast<int>(
      std::min<int64_t>(kThreads / g, std::max<int64_t>(1, (rows + sms - 1) / sms)));
  if (g < 32) p.per_block = (p.per_block + 32 / g - 1) / (32 / g) * (32 / g);  // whole warps
  const int64_t need = std::max<int64_t>(1, (rows + p.per_block - 1) / p.per_block);
  int most = sms;
  while (most > 1 && need > most && (static_cast<int64_t>(most) * p.per_block) % v != 0) --most;
  p.blocks = static_cast<int>(std::min<int64_t>(need, most));
  return p;
}

// Whether rows of `n` dense elements can be read as shifted vectors of V.
template <typename T, int V>
bool shifted_rows(const void* p, int64_t stride, int64_t n) {
  return shift_fits(n, V) && stride == n && vec_rows<T, V>(p, 0, V);
}

unsigned row_blocks(int64_t rows) {
  const int64_t blocks = (rows + 7) / 8;
  return static_cast<unsigned>(std::min<int64_t>(blocks, device_sm_count() * 8));
}

template <typename Tx, typename Tw, typename Ty, int V, int VPT>
int forward_held(const NormForward& a, int g, cudaStream_t stream) {
  const int threads = g > 32 ? g : 256;
  const int64_t per_block = g > 32 ? 1 : threads / g;
  const int64_t blocks = (a.rows + per_block - 1) / per_block;
  return launched(
      launch_kernel(norm_forward_held<Tx, Tw, Ty, V, VPT>, dim3(static_cast<unsigned>(blocks)),
                    dim3(threads), 0, stream, 1, static_cast<const Tx*>(a.x), a.x_stride,
                    static_cast<const Tw*>(a.weight), static_cast<const Tw*>(a.bias), a.eps,
                    static_cast<Ty*>(a.y), a.mean, a.rstd, a.rows, static_cast<int>(a.features), g),
      "layer norm forward");
}

// 16 bytes of x per load where every row allows it, else single elements.
template <typename Tx>
constexpr int kWide = 16 / sizeof(Tx);

template <auto KERNEL, typename... Args>
int launch_ring(const Rings& p, size_t smem, cudaStream_t stream, const char* what, Args... args) {
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
  });
  if (e != cudaSuccess) return cuda_error(e, what);
  return launched(launch_kernel(KERNEL, dim3(p.blocks), dim3(p.per_block * p.g), smem, stream, 1,
                                args...),
                  what);
}

template <typename Tx, typename Tw, typename Ty>
struct RunForward {
  static constexpr int V = kWide<Tx>;
  template <int W, bool SHIFT>
  static int ring(const NormForward& a, cudaStream_t stream) {
    constexpr int bytes = Held<Tx, W>::kBytes;
    const int g = group_size(a.features + (SHIFT ? W - 1 : 0), kHeld, kThreads);
    const Rings p = plan_rings(a.rows, g, SHIFT ? W : 1);
    const size_t smem = static_cast<size_t>(p.per_block) * g * bytes * kRingStages<bytes>;
    return launch_ring<norm_forward_ring<Tx, Tw, Ty, W, SHIFT>>(
        p, smem, stream, "layer norm forward", static_cast<const Tx*>(a.x), a.x_stride,
        static_cast<const Tw*>(a.weight), static_cast<const Tw*>(a.bias), a.eps,
        static_cast<Ty*>(a.y), a.mean, a.rstd, a.rows, static_cast<int>(a.features), g);
  }
  template <int W>
  static int held(const NormForward& a, cudaStream_t stream) {
    // 32 elements per thread keep 513 to 1024 features within a warp (no
    // block-wide sum) and reach the widest rows.
    const int64_t d = a.features;
    if ((d > 512 && d <= 1024) || d > 16384) {
      return forward_held<Tx, Tw, Ty, W, 32 / W>(a, group_size(d, 32, 1024), stream);
    }
    return forward_held<Tx, Tw, Ty, W, 16 / W>(a, group_size(d, 16, 1024), stream);
  }
  static int run(const NormForward& a, cudaStream_t stream) {
    const bool wide = vec_rows<Tx, V>(a.x, a.x_stride, a.features) &&
                      vec_rows<Ty, V>(a.y, a.features, a.features);
    if (a.features <= kThreads * kHeld) {
      if (wide) return ring<V, false>(a, stream);
      if (vec_rows<Tx, 2>(a.x, a.x_stride, a.features) &&
          vec_rows<Ty, 2>(a.y, a.features, a.features)) {
        return ring<2, false>(a, stream);
      }
      if (a.features + V - 1 <= kThreads * kHeld &&
          shifted_rows<Tx, V>(a.x, a.x_stride, a.features) &&
          shifted_rows<Ty, V>(a.y, a.features, a.features)) {
        return ring<V, true>(a, stream);
      }
    }
    if (a.features <= 32768) {
      return wide && vec_rows<Tw, V>(a.weight, 0, V) && vec_rows<Tw, V>(a.bias, 0, V)
                 ? held<V>(a, stream)
                 : held<1>(a, stream);
    }
    return launched(
        launch_kernel(norm_forward_rows<Tx, Tw, Ty>, dim3(row_blocks(a.rows)), dim3(256), 0, stream,
                      1, static_cast<const Tx*>(a.x), a.x_stride, static_cast<const Tw*>(a.weight),
                      static_cast<const Tw*>(a.bias), a.eps, static_cast<Ty*>(a.y), a.mean, a.rstd,
                      a.rows, a.features),
        "layer norm forward");
  }
};

template <typename Tx, typename Tw, typename Ty>
struct RunBackward {
  static constexpr int V = kWide<Tx>;
  template <int W, bool SHIFT>
  static int ring(const NormBackward& a, float* partial, int* slices, cudaStream_t stream) {
    constexpr int bytes = Held<Tx, W>::kBytes + Held<Ty, W>::kBytes;
    const int g = group_size(a.features + (SHIFT ? W - 1 : 0), kHeld, kThreads);
    const Rings p = plan_rings(a.rows, g, SHIFT ? W : 1);
    *slices = p.blocks;
    const size_t sums = static_cast<size_t>(p.per_block) * 2 * a.features * sizeof(float);
    const size_t stages =
        W > 1 ? static_cast<size_t>(p.per_block) * g * bytes * kRingStages<bytes> : 0;
    return launch_ring<norm_backward_ring<Tx, Tw, Ty, W, SHIFT>>(
        p, std::max(sums, stages), stream, "layer norm backward", static_cast<const Ty*>(a.dy),
        a.dy_stride, static_cast<const Tx*>(a.x), a.x_stride, a.mean, a.rstd,
        static_cast<const Tw*>(a.weight), static_cast<Tx*>(a.dx), partial, a.rows,
        static_cast<int>(a.features), g);
  }
  static int run(const NormBackward& a, void* ws, cudaStream_t stream) {
    float* partial = static_cast<float*>(ws);
    const Ty* dy = static_cast<const Ty*>(a.dy);
    const Tx* x = static_cast<const Tx*>(a.x);
    const int64_t d = a.features;
    int slices = 0;
    int rc = CCV_OK;
    if (d <= kThreads * kHeld) {
      if (vec_rows<Tx, V>(x, a.x_stride, d) && vec_rows<Ty, V>(dy, a.dy_stride, d) &&
          vec_rows<Tx, V>(a.dx, d, d)) {
        rc = ring<V, false>(a, partial, &slices, stream);
      } else if (vec_rows<Tx, 2>(x, a.x_stride, d) && vec_rows<Ty, 2>(dy, a.dy_stride, d) &&
                 vec_rows<Tx, 2>(a.dx, d, d)) {
        rc = ring<2, false>(a, partial, &slices, stream);
      } else if (d + V - 1 <= kThreads * kHeld && shifted_rows<Tx, V>(x, a.x_stride, d) &&
                 shifted_rows<Ty, V>(dy, a.dy_stride, d) && shifted_rows<Tx, V>(a.dx, d, d)) {
        rc = ring<V, true>(a, partial, &slices, stream);
      } else {
        rc = ring<1, false>(a, partial, &slices, stream);
      }
    } else {
      slices = column_slices(a.rows);
      if (a.dx != nullptr && a.rows > 0) {
        rc = launched(launch_kernel(norm_backward_rows<Tx, Tw, Ty>, dim3(row_blocks(a.rows)),
                                    dim3(256), 0, stream, 1, dy, a.dy_stride, x, a.x_stride, a.mean,
                                    a.rstd, static_cast<const Tw*>(a.weight),
                                    static_cast<Tx*>(a.dx), a.rows, a.features),
                      "layer norm backward");
      }
      if (rc == CCV_OK) {
        const unsigned cols =
            static_cast<unsigned>((a.features + kColThreadsX - 1) / kColThreadsX);
        rc = launched(launch_kernel(norm_backward_columns<Tx, Ty>, dim3(cols, slices),
                                    dim3(kColThreadsX, kColThreadsY), 0, stream, 1, dy, a.dy_stride,
                                    x, a.x_stride, a.mean, a.rstd, partial, a.rows, a.features),
                      "layer norm backward columns");
      }
    }
    if (rc != CCV_OK || (a.dweight == nullptr && a.dbias == nullptr)) return rc;
    return launched(
        launch_kernel(norm_backward_reduce<Tw>,
                      dim3(static_cast<unsigned>((a.features + 31) / 32)), dim3(1024), 0, stream, 1,
                      static_cast<const float*>(partial), slices, static_cast<Tw*>(a.dweight),
                      static_cast<Tw*>(a.dbias), a.features),
        "layer norm backward reduce");
  }
};

// Calls Run<Tx, Tw, Ty>::run for the types of a call (the valid combinations
// only; the entry points reject the others).
template <template <typename, typename, typename> class Run, typename T16, typename... Args>
int dispatch16(int weight_dtype, int y_dtype, Args&&... args) {
  const bool w32 = weight_dtype == CCV_DTYPE_F32, y32 = y_dtype == CCV_DTYPE_F32;
  if (w32 && y32) return Run<T16, float, float>::run(args...);
  if (w32) return Run<T16, float, T16>::run(args...);
  if (y32) return Run<T16, T16, float>::run(args...);
  return Run<T16, T16, T16>::run(args...);
}
template <template <typename, typename, typename> class Run, typename... Args>
int dispatch(int x_dtype, int weight_dtype, int y_dtype, Args&&... args) {
  if (x_dtype == CCV_DTYPE_BF16) {
    return dispatch16<Run, __nv_bfloat16>(weight_dtype, y_dtype, args...);
  }
  if (x_dtype == CCV_DTYPE_F16) return dispatch16<Run, __half>(weight_dtype, y_dtype, args...);
  if (y_dtype == CCV_DTYPE_BF16) return Run<float, float, __nv_bfloat16>::run(args...);
  if (y_dtype == CCV_DTYPE_F16) return Run<float, float, __half>::run(args...);
  return Run<float, float, float>::run(args...);
}

}  // namespace

size_t norm_backward_workspace_bytes(int64_t rows, int64_t features) {
  // Blocks of the ring kernels, or slices of the wide rows' column sums.
  const int64_t slices =
      std::max<int64_t>(std::min<int64_t>(std::max<int64_t>(rows, 1), device_sm_count()),
                        column_slices(rows));
  return static_cast<size_t>(slices) * 2 * static_cast<size_t>(features) * sizeof(float);
}

int launch_norm_forward(const NormForward& a, cudaStream_t stream) {
  return dispatch<RunForward>(a.x_dtype, a.weight_dtype, a.y_dtype, a, stream);
}

int launch_norm_backward(const NormBackward& a, void* ws, cudaStream_t stream) {
  return dispatch<RunBackward>(a.x_dtype, a.weight_dtype, a.y_dtype, a, ws, stream);
}

}  // namespace ccv
