// Layer norm over rows of features, forward and backward.
//
//   mean = sum_j x_j / D,  var = sum_j (x_j - mean)^2 / D,  r = 1/sqrt(var + eps)
//   y_j = (x_j - mean) r w_j + b_j
// and with z_j = (x_j - mean) r, t_j = dy_j w_j:
//   dx_j = r (t_j - sum t / D - z_j sum(t z) / D)
//   dw_j = sum_rows dy_j z_j,   db_j = sum_rows dy_j
//
// Both directions are bound by memory: the forward pass reads x and writes y
// once, the backward pass reads x and dy and writes dx once.  A group of G
// threads holds a row in registers, so the mean, the centred squares and the
// output come from one read; G is the fewest threads (a power of two within
// a warp, then whole warps) that hold the row at 16 or 32 elements each, so
// narrow rows share a warp and few shuffles are spent per element.  The
// backward pass keeps each thread's columns fixed and sums dw and db over the
// rows in registers, reading nothing twice; blocks leave fp32 partial sums
// that a second launch adds in block order (deterministic).  Rows too wide
// for a block's registers take kernels that read them again from the caches.
#include <algorithm>

#include "ccv_internal.h"
#include "ccv_ptx.cuh"
#include "ccv_tokens.cuh"

namespace ccv {

namespace {

// Sum over the G threads of a row's group: shuffles within a warp, then
// (G > 32: the group is the block) one exchange through shared memory, in
// warp order.  `red` holds 32 entries per call in flight; successive calls
// alternate between two of them.
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

// Forward, rows in registers: VPT vectors of V elements per thread.
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

constexpr int kBackwardThreads = 512;  // most threads of a backward block
constexpr int kBackwardHeld = 16;      // elements per thread

// Backward, rows in registers; partial: [blocks][2][features].
template <typename Tx, typename Tw, typename Ty, int V>
__global__ void __launch_bounds__(kBackwardThreads, 1)
    norm_backward_held(const Ty* __restrict__ dy, int64_t dy_stride, const Tx* __restrict__ x,
                       int64_t x_stride, const float* __restrict__ mean_in,
                       const float* __restrict__ rstd_in, const Tw* __restrict__ w,
                       Tx* __restrict__ dx, float* __restrict__ partial, int64_t rows,
                       int features, int g) {
  constexpr int VPT = kBackwardHeld / V;
  __shared__ float red[2][kBackwardThreads / 32][2];
  extern __shared__ float columns[];  // [2][features], g <= 32
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const bool wide = g > 32;
  const int lane = wide ? threadIdx.x : threadIdx.x & (g - 1);
  const int per_block = wide ? 1 : blockDim.x / g;
  const int group = wide ? 0 : threadIdx.x / g;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
  const float inv = 1.f / static_cast<float>(features);
  float wt[VPT][V], dw[VPT][V] = {}, db[VPT][V] = {};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (i * g + lane) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) wt[i][j] = 1.f;
    if (w != nullptr && c < features) {
      const Vec<Tw, V> wv = load_vec<Tw, V>(w + c);
#pragma unroll
      for (int j = 0; j < V; ++j) wt[i][j] = to_f32(wv.e[j]);
    }
  }
  Vec<Tx, V> rx[VPT];
  Vec<Ty, V> rg[VPT];
  float mean = 0.f, rstd = 0.f;
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * g + lane) * V;
      if (c < features) {
        rx[i] = load_vec<Tx, V>(x + r * x_stride + c);
        rg[i] = load_vec<Ty, V>(dy + r * dy_stride + c);
      }
    }
    mean = mean_in[r];
    rstd = rstd_in[r];
  };
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per_block;
  if (first + group < rows) fetch(first + group);
  int parity = 0;
  // The block's groups walk together: every thread takes part in each sum.
  for (int64_t r0 = first; r0 < rows; r0 += step, parity ^= 1) {
    const int64_t r = r0 + group;
    const bool live = r < rows;
    float z[VPT][V], t[VPT][V];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const bool in = live && (i * g + lane) * V < features;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        z[i][j] = 0.f;
        t[i][j] = 0.f;
        if (in) {
          const float d = to_f32(rg[i].e[j]);
          z[i][j] = (to_f32(rx[i].e[j]) - mean) * rstd;
          t[i][j] = d * wt[i][j];
          dw[i][j] = fmaf(d, z[i][j], dw[i][j]);
          db[i][j] += d;
          sum[0] += t[i][j];
          sum[1] = fmaf(t[i][j], z[i][j], sum[1]);
        }
      }
    }
    const float scale = rstd;
    // The next row's loads are in flight during this row's sums and stores.
    if (r + step < rows) fetch(r + step);
    group_sum<2>(sum, g, red[parity]);
    if (live && dx != nullptr) {
      const float a = sum[0] * inv, c1 = sum[1] * inv;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = (i * g + lane) * V;
        if (c < features) {
          float o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = scale * (t[i][j] - a - z[i][j] * c1);
          store_vec<Tx, V>(dx + r * features + c, o);
        }
      }
    }
  }
  float* out = partial + static_cast<int64_t>(blockIdx.x) * 2 * features;
  if (wide) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * g + lane) * V;
      if (c < features) {
        store_vec<float, V>(out + c, dw[i]);
        store_vec<float, V>(out + features + c, db[i]);
      }
    }
    return;
  }
  // Groups that share a warp add up by shuffles, the warps in turn.
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      for (int o = 16; o >= g; o >>= 1) {
        dw[i][j] += __shfl_xor_sync(0xffffffffu, dw[i][j], o);
        db[i][j] += __shfl_xor_sync(0xffffffffu, db[i][j], o);
      }
    }
  }
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int k = 0; k < warps; ++k) {
    if (warp == k && (threadIdx.x & 31) < g) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = (i * g + lane) * V + j;
          if (c < features) {
            columns[c] = k == 0 ? dw[i][j] : columns[c] + dw[i][j];
            columns[features + c] = k == 0 ? db[i][j] : columns[features + c] + db[i][j];
          }
        }
      }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < 2 * features; c += blockDim.x) out[c] = columns[c];
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
// columns per block, eight warps take every eighth slice, then add up in
// warp order.
template <typename Tw>
__global__ void __launch_bounds__(256) norm_backward_reduce(const float* __restrict__ partial,
                                                            int slices, Tw* __restrict__ dw,
                                                            Tw* __restrict__ db,
                                                            int64_t features) {
  __shared__ float sh[2][8][32];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sw = 0.f, sb = 0.f;
  if (j < features) {
#pragma unroll 4
    for (int s = warp; s < slices; s += 8) {
      sw += partial[(static_cast<int64_t>(s) * 2) * features + j];
      sb += partial[(static_cast<int64_t>(s) * 2 + 1) * features + j];
    }
  }
  sh[0][warp][lane] = sw;
  sh[1][warp][lane] = sb;
  __syncthreads();
  if (warp < 2 && j < features) {
    Tw* out = warp == 0 ? dw : db;
    if (out != nullptr) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) v += sh[warp][k][lane];
      out[j] = from_f32<Tw>(v);
    }
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

int64_t backward_blocks(int64_t rows) {
  // Two blocks of up to 256 threads per SM (128 registers each).
  return std::max<int64_t>(1, std::min<int64_t>(rows, 2 * device_sm_count()));
}

unsigned row_blocks(int64_t rows) {
  const int64_t blocks = (rows + 7) / 8;
  return static_cast<unsigned>(blocks < 148 * 8 ? blocks : 148 * 8);
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

template <typename Tx, typename Tw, typename Ty>
struct RunForward {
  template <int V>
  static int held(const NormForward& a, cudaStream_t stream) {
    // 32 elements per thread keep 513 to 1024 features within a warp (no
    // block-wide sum) and reach the widest rows.
    const int64_t d = a.features;
    if ((d > 512 && d <= 1024) || d > 16384) {
      return forward_held<Tx, Tw, Ty, V, 32 / V>(a, group_size(d, 32, 1024), stream);
    }
    return forward_held<Tx, Tw, Ty, V, 16 / V>(a, group_size(d, 16, 1024), stream);
  }
  static int run(const NormForward& a, cudaStream_t stream) {
    constexpr int V = kWide<Tx>;
    if (a.features <= 32768) {
      if (vec_rows<Tx, V>(a.x, a.x_stride, a.features) &&
          vec_rows<Ty, V>(a.y, a.features, a.features) &&
          vec_rows<Tw, V>(a.weight, 0, a.features) && vec_rows<Tw, V>(a.bias, 0, a.features)) {
        return held<V>(a, stream);
      }
      return held<1>(a, stream);
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
  template <int V>
  static int held(const NormBackward& a, int g, int64_t blocks, float* partial,
                  cudaStream_t stream) {
    const size_t smem = g > 32 ? 0 : static_cast<size_t>(a.features) * 2 * sizeof(float);
    return launched(
        launch_kernel(norm_backward_held<Tx, Tw, Ty, V>, dim3(static_cast<unsigned>(blocks)),
                      dim3(g > 32 ? g : 256), smem, stream, 1, static_cast<const Ty*>(a.dy),
                      a.dy_stride, static_cast<const Tx*>(a.x), a.x_stride, a.mean, a.rstd,
                      static_cast<const Tw*>(a.weight), static_cast<Tx*>(a.dx), partial, a.rows,
                      static_cast<int>(a.features), g),
        "layer norm backward");
  }
  static int run(const NormBackward& a, void* ws, cudaStream_t stream) {
    constexpr int V = kWide<Tx>;
    float* partial = static_cast<float*>(ws);
    const Ty* dy = static_cast<const Ty*>(a.dy);
    const Tx* x = static_cast<const Tx*>(a.x);
    const int g = group_size(a.features, kBackwardHeld, kBackwardThreads);
    int slices;
    int rc = CCV_OK;
    if (g > 0) {
      const int64_t per_block = g > 32 ? 1 : 256 / g;
      const int64_t blocks = backward_blocks((a.rows + per_block - 1) / per_block);
      slices = static_cast<int>(blocks);
      const bool wide = vec_rows<Tx, V>(x, a.x_stride, a.features) &&
                        vec_rows<Ty, V>(dy, a.dy_stride, a.features) &&
                        vec_rows<Tx, V>(a.dx, a.features, a.features) &&
                        vec_rows<Tw, V>(a.weight, 0, a.features);
      rc = wide ? held<V>(a, g, blocks, partial, stream) : held<1>(a, g, blocks, partial, stream);
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
                      dim3(static_cast<unsigned>((a.features + 31) / 32)), dim3(256), 0, stream, 1,
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
  const int64_t slices = group_size(features, kBackwardHeld, kBackwardThreads) > 0
                             ? backward_blocks(rows)
                             : column_slices(rows);
  return static_cast<size_t>(slices) * 2 * static_cast<size_t>(features) * sizeof(float);
}

int launch_norm_forward(const NormForward& a, cudaStream_t stream) {
  return dispatch<RunForward>(a.x_dtype, a.weight_dtype, a.y_dtype, a, stream);
}

int launch_norm_backward(const NormBackward& a, void* ws, cudaStream_t stream) {
  return dispatch<RunBackward>(a.x_dtype, a.weight_dtype, a.y_dtype, a, ws, stream);
}

}  // namespace ccv
