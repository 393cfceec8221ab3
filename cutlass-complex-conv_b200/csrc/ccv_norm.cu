// Layer norm over rows of features, forward and backward.
//
//   mean = sum_j x_j / D,  var = sum_j (x_j - mean)^2 / D,  r = 1/sqrt(var + eps)
//   y_j = (x_j - mean) r w_j + b_j
// and with z_j = (x_j - mean) r, t_j = dy_j w_j:
//   dx_j = r (t_j - sum t / D - z_j sum(t z) / D)
//   dw_j = sum_rows dy_j z_j,   db_j = sum_rows dy_j
#include "ccv_internal.h"
#include "ccv_ptx.cuh"
#include "ccv_tokens.cuh"

namespace ccv {

namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp per row; the row is read three times (from L1/L2 after the first).
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

// Column sums over one slice of rows: partial [slices][2][features].
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

// dweight and dbias from the slices' partial sums, added in slice order.
template <typename Tw>
__global__ void norm_backward_reduce(const float* __restrict__ partial, int slices,
                                     Tw* __restrict__ dw, Tw* __restrict__ db, int64_t features) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int64_t j = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (j >= features) return;
  float sw = 0.f, sb = 0.f;
  for (int s = 0; s < slices; ++s) {
    sw += partial[(static_cast<int64_t>(s) * 2) * features + j];
    sb += partial[(static_cast<int64_t>(s) * 2 + 1) * features + j];
  }
  if (dw != nullptr) dw[j] = from_f32<Tw>(sw);
  if (db != nullptr) db[j] = from_f32<Tw>(sb);
}

int column_slices(int64_t rows) {
  const int64_t s = (rows + 63) / 64;
  return static_cast<int>(s < 1 ? 1 : (s > 128 ? 128 : s));
}

}  // namespace

size_t norm_backward_workspace_bytes(int64_t rows, int64_t features) {
  return static_cast<size_t>(column_slices(rows)) * 2 * static_cast<size_t>(features) *
         sizeof(float);
}

namespace {

unsigned row_blocks(int64_t rows) {
  const int64_t blocks = (rows + 7) / 8;
  return static_cast<unsigned>(blocks < 148 * 8 ? blocks : 148 * 8);
}

template <typename Tx, typename Tw, typename Ty>
struct RunForward {
  static int run(const NormForward& a, cudaStream_t stream) {
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
  static int run(const NormBackward& a, void* ws, cudaStream_t stream) {
    const int slices = column_slices(a.rows);
    float* partial = static_cast<float*>(ws);
    const Ty* dy = static_cast<const Ty*>(a.dy);
    const Tx* x = static_cast<const Tx*>(a.x);
    int rc = CCV_OK;
    if (a.dx != nullptr && a.rows > 0) {
      rc = launched(launch_kernel(norm_backward_rows<Tx, Tw, Ty>, dim3(row_blocks(a.rows)),
                                  dim3(256), 0, stream, 1, dy, a.dy_stride, x, a.x_stride, a.mean,
                                  a.rstd, static_cast<const Tw*>(a.weight), static_cast<Tx*>(a.dx),
                                  a.rows, a.features),
                    "layer norm backward");
      if (rc != CCV_OK) return rc;
    }
    if (a.dweight == nullptr && a.dbias == nullptr) return CCV_OK;
    const unsigned cols = static_cast<unsigned>((a.features + kColThreadsX - 1) / kColThreadsX);
    rc = launched(launch_kernel(norm_backward_columns<Tx, Ty>, dim3(cols, slices),
                                dim3(kColThreadsX, kColThreadsY), 0, stream, 1, dy, a.dy_stride, x,
                                a.x_stride, a.mean, a.rstd, partial, a.rows, a.features),
                  "layer norm backward columns");
    if (rc != CCV_OK) return rc;
    return launched(
        launch_kernel(norm_backward_reduce<Tw>,
                      dim3(static_cast<unsigned>((a.features + 127) / 128)), dim3(128), 0, stream,
                      1, static_cast<const float*>(partial), slices, static_cast<Tw*>(a.dweight),
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

int launch_norm_forward(const NormForward& a, cudaStream_t stream) {
  return dispatch<RunForward>(a.x_dtype, a.weight_dtype, a.y_dtype, a, stream);
}

int launch_norm_backward(const NormBackward& a, void* ws, cudaStream_t stream) {
  return dispatch<RunBackward>(a.x_dtype, a.weight_dtype, a.y_dtype, a, ws, stream);
}

}  // namespace ccv
