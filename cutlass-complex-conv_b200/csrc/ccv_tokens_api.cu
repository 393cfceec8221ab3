// extern "C" entry points of the token operators (declared in
// include/ccv_b200.h): argument checks, then the launchers.  No C++ exception
// leaves them.
#include <cmath>
#include <exception>

#include "ccv_internal.h"
#include "ccv_tokens.cuh"

namespace ccv {
namespace {

// Runs body(), turning an exception (an allocation of an error text) into a
// status.
template <typename Fn>
int guarded(Fn&& body) noexcept {
  try {
    return body();
  } catch (...) {
    return CCV_ERR_CUDA;
  }
}

// The same for a size query: 0 when it cannot be answered.
template <typename Fn>
size_t guarded_size(Fn&& body) noexcept {
  try {
    return body();
  } catch (...) {
    return 0;
  }
}

int invalid(const char* msg) { return set_error(CCV_ERR_INVALID_ARGUMENT, msg); }

bool aligned_to(const void* p, size_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

constexpr int64_t kMaxExtent = 0x7fffffffLL;
constexpr int64_t kMaxElements = 1LL << 40;

int check_rows(int64_t rows, int64_t features) {
  if (rows < 0) return invalid("rows must be non-negative");
  if (features <= 0) return invalid("features must be positive");
  if (rows > kMaxExtent || features > kMaxExtent || rows * features > kMaxElements) {
    return set_error(CCV_ERR_UNSUPPORTED, "tensor too large");
  }
  return CCV_OK;
}

int check_norm_types(int x_dtype, int weight_dtype, int y_dtype) {
  if (!valid_dtype(x_dtype) || !valid_dtype(weight_dtype) || !valid_dtype(y_dtype)) {
    return invalid("unknown element type");
  }
  if (weight_dtype != CCV_DTYPE_F32 && weight_dtype != x_dtype) {
    return invalid("layer norm weights must be float32 or of the input's type");
  }
  if (x_dtype != CCV_DTYPE_F32 && y_dtype != CCV_DTYPE_F32 && y_dtype != x_dtype) {
    return invalid("a 16-bit input gives an output of its own type or float32");
  }
  return CCV_OK;
}

int check_ffn(const FfnShape& s) {
  if (s.dtype != CCV_DTYPE_BF16 && s.dtype != CCV_DTYPE_F16) {
    return invalid("the gated feed-forward block takes bfloat16 or float16");
  }
  if (s.activation != CCV_ACTIVATION_SILU && s.activation != CCV_ACTIVATION_GELU) {
    return invalid("unknown activation");
  }
  if (s.hidden <= 0) return invalid("hidden must be positive");
  int rc = check_rows(s.rows, s.features);
  if (rc == CCV_OK) rc = check_rows(s.rows, s.hidden);
  if (rc == CCV_OK) rc = check_rows(s.hidden, s.features);
  return rc;
}

// Rows of `length` elements that TMA reads in place (see FfnForward).
int check_in_place(const void* p, int64_t length, int64_t stride, const char* msg) {
  if (length % 8 == 0 && (!aligned_to(p, 16) || stride % 8 != 0)) return invalid(msg);
  return CCV_OK;
}

int check_ffn_alignment(const FfnShape& s, const void* x, int64_t x_stride, const void* w_gate,
                        const void* w_up, const void* w_down) {
  const char* msg = "rows of a multiple of 8 elements must start at 16-byte boundaries";
  int rc = check_in_place(x, s.features, s.rows > 1 ? x_stride : 0, msg);
  if (rc == CCV_OK) rc = check_in_place(w_gate, s.features, 0, msg);
  if (rc == CCV_OK) rc = check_in_place(w_up, s.features, 0, msg);
  return rc == CCV_OK ? check_in_place(w_down, s.hidden, 0, msg) : rc;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  if (need == 0) return CCV_OK;
  if (ws == nullptr || !aligned_to(ws, 256) || have < need) {
    return set_error(CCV_ERR_WORKSPACE, "workspace missing, misaligned or too small");
  }
  return CCV_OK;
}

// Checks of both dropout entries and the launch; `types`: what to say of two
// 16-bit types that differ.
int run_dropout(const Dropout& a, const char* types, ccv_stream_t stream) {
  if (!valid_dtype(a.x_dtype) || !valid_dtype(a.y_dtype)) return invalid("unknown element type");
  if (a.count < 0) return invalid("count must be non-negative");
  if (a.count > kMaxElements) return set_error(CCV_ERR_UNSUPPORTED, "tensor too large");
  if (!(a.p >= 0.0 && a.p <= 1.0)) return invalid("p must be between 0 and 1");
  if (a.x_dtype != CCV_DTYPE_F32 && a.y_dtype != CCV_DTYPE_F32 && a.y_dtype != a.x_dtype) {
    return invalid(types);
  }
  if (a.count == 0) return CCV_OK;
  if (a.x == nullptr || a.y == nullptr) return invalid("null tensor pointer");
  if (!aligned_to(a.x, dtype_bytes(a.x_dtype)) || !aligned_to(a.y, dtype_bytes(a.y_dtype)) ||
      !aligned_to(a.residual, dtype_bytes(a.y_dtype)) || !aligned_to(a.offset_dev, 8)) {
    return invalid("tensor pointers must be aligned to their element");
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int rc = begin_launches(st);
  return rc != CCV_OK ? rc : launch_dropout(a, st);
}

}  // namespace
}  // namespace ccv

using namespace ccv;

extern "C" {

int ccv_layer_norm_forward(const void* x, int x_dtype, int64_t x_row_stride, const void* weight,
                           const void* bias, int weight_dtype, float eps, void* y, int y_dtype,
                           float* mean, float* rstd, int64_t rows, int64_t features,
                           ccv_stream_t stream) {
  return guarded([&]() -> int {
    int rc = check_rows(rows, features);
    if (rc == CCV_OK) rc = check_norm_types(x_dtype, weight_dtype, y_dtype);
    if (rc != CCV_OK) return rc;
    if (!(eps >= 0.f) || std::isinf(eps)) return invalid("eps must be non-negative and finite");
    if (rows == 0) return CCV_OK;
    if (x == nullptr || y == nullptr) return invalid("null tensor pointer");
    if (x_row_stride < 0) return invalid("row stride must be non-negative");
    if (!aligned_to(x, dtype_bytes(x_dtype)) || !aligned_to(y, dtype_bytes(y_dtype)) ||
        !aligned_to(weight, dtype_bytes(weight_dtype)) ||
        !aligned_to(bias, dtype_bytes(weight_dtype)) || !aligned_to(mean, 4) ||
        !aligned_to(rstd, 4)) {
      return invalid("tensor pointers must be aligned to their element");
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if ((rc = begin_launches(st)) != CCV_OK) return rc;
    NormForward a = {x,    x_row_stride, weight,  bias,         eps,    y, mean, rstd, rows,
                     features, x_dtype,  weight_dtype, y_dtype};
    return launch_norm_forward(a, st);
  });
}

size_t ccv_layer_norm_backward_workspace_bytes(int64_t rows, int64_t features) {
  return guarded_size([&]() -> size_t {
    return check_rows(rows, features) == CCV_OK ? norm_backward_workspace_bytes(rows, features) : 0;
  });
}

int ccv_layer_norm_backward(const void* dy, int y_dtype, int64_t dy_row_stride, const void* x,
                            int x_dtype, int64_t x_row_stride, const float* mean,
                            const float* rstd, const void* weight, int weight_dtype, void* dx,
                            void* dweight, void* dbias, int64_t rows, int64_t features,
                            void* workspace, size_t workspace_bytes, ccv_stream_t stream) {
  return guarded([&]() -> int {
    int rc = check_rows(rows, features);
    if (rc == CCV_OK) rc = check_norm_types(x_dtype, weight_dtype, y_dtype);
    if (rc != CCV_OK) return rc;
    if (dx == nullptr && dweight == nullptr && dbias == nullptr) return CCV_OK;
    if (rows > 0 && (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr)) {
      return invalid("null tensor pointer");
    }
    if (x_row_stride < 0 || dy_row_stride < 0) return invalid("row stride must be non-negative");
    if (!aligned_to(x, dtype_bytes(x_dtype)) || !aligned_to(dx, dtype_bytes(x_dtype)) ||
        !aligned_to(dy, dtype_bytes(y_dtype)) || !aligned_to(weight, dtype_bytes(weight_dtype)) ||
        !aligned_to(dweight, dtype_bytes(weight_dtype)) ||
        !aligned_to(dbias, dtype_bytes(weight_dtype)) || !aligned_to(mean, 4) ||
        !aligned_to(rstd, 4)) {
      return invalid("tensor pointers must be aligned to their element");
    }
    if ((rc = check_workspace(workspace, workspace_bytes,
                              norm_backward_workspace_bytes(rows, features))) != CCV_OK) {
      return rc;
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if ((rc = begin_launches(st)) != CCV_OK) return rc;
    NormBackward a = {dy, dy_row_stride, x,     x_row_stride, mean,     rstd,    weight,      dx,
                      dweight, dbias,    rows,  features,     x_dtype,  weight_dtype, y_dtype};
    return launch_norm_backward(a, workspace, st);
  });
}

size_t ccv_gated_ffn_saved_bytes(int64_t rows, int64_t features, int64_t hidden) {
  const FfnShape s = {rows, features, hidden, CCV_DTYPE_BF16, 0};
  return guarded_size(
      [&]() -> size_t { return check_ffn(s) == CCV_OK ? ffn_saved_planes(s) * ffn_plane_bytes(s) : 0; });
}

size_t ccv_gated_ffn_forward_workspace_bytes(int64_t rows, int64_t features, int64_t hidden,
                                             int save) {
  const FfnShape s = {rows, features, hidden, CCV_DTYPE_BF16, 0};
  return guarded_size([&]() -> size_t {
    return check_ffn(s) == CCV_OK ? ffn_forward_workspace_bytes(s, save != 0) : 0;
  });
}

size_t ccv_gated_ffn_backward_workspace_bytes(int64_t rows, int64_t features, int64_t hidden) {
  const FfnShape s = {rows, features, hidden, CCV_DTYPE_BF16, 0};
  return guarded_size([&]() -> size_t {
    return check_ffn(s) == CCV_OK ? ffn_backward_workspace_bytes(s) : 0;
  });
}

int ccv_gated_ffn_forward(const void* x, int64_t x_row_stride, const void* w_gate,
                          const void* w_up, const void* w_down, void* y, int dtype,
                          int activation, int64_t rows, int64_t features, int64_t hidden,
                          void* saved, size_t saved_bytes, void* workspace,
                          size_t workspace_bytes, ccv_stream_t stream) {
  return guarded([&]() -> int {
    FfnForward f = {{rows, features, hidden, dtype, activation},
                    x, rows > 1 ? x_row_stride : features, w_gate, w_up, w_down, y, saved};
    int rc = check_ffn(f.shape);
    if (rc != CCV_OK || rows == 0) return rc;
    if (x == nullptr || w_gate == nullptr || w_up == nullptr || w_down == nullptr ||
        y == nullptr) {
      return invalid("null tensor pointer");
    }
    if (rows > 1 && x_row_stride < features) return invalid("row stride below the row length");
    for (const void* p : {x, w_gate, w_up, w_down, static_cast<const void*>(y)}) {
      if (!aligned_to(p, 2)) return invalid("tensor pointers must be aligned to their element");
    }
    if ((rc = check_ffn_alignment(f.shape, x, x_row_stride, w_gate, w_up, w_down)) != CCV_OK ||
        (rc = check_in_place(y, features, 0, "y must be 16-byte aligned")) != CCV_OK) {
      return rc;
    }
    if (saved != nullptr && (!aligned_to(saved, 256) || saved_bytes < ffn_saved_planes(f.shape) * ffn_plane_bytes(f.shape))) {
      return set_error(CCV_ERR_WORKSPACE, "saved buffer misaligned or too small");
    }
    if ((rc = check_workspace(workspace, workspace_bytes,
                              ffn_forward_workspace_bytes(f.shape, saved != nullptr))) != CCV_OK) {
      return rc;
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if ((rc = begin_launches(st)) != CCV_OK) return rc;
    return launch_ffn_forward(f, workspace, st);
  });
}

int ccv_gated_ffn_backward(const void* dy, int64_t dy_row_stride, const void* x,
                           int64_t x_row_stride, const void* w_gate, const void* w_up,
                           const void* w_down, const void* saved, size_t saved_bytes, void* dx,
                           void* dw_gate, void* dw_up, void* dw_down, int dtype, int activation,
                           int64_t rows, int64_t features, int64_t hidden, void* workspace,
                           size_t workspace_bytes, ccv_stream_t stream) {
  return guarded([&]() -> int {
    FfnBackward b = {{rows, features, hidden, dtype, activation},
                     dy, rows > 1 ? dy_row_stride : features,
                     x, rows > 1 ? x_row_stride : features, w_gate, w_up, w_down, saved,
                     dx, dw_gate, dw_up, dw_down};
    int rc = check_ffn(b.shape);
    if (rc != CCV_OK) return rc;
    if (dx == nullptr && dw_gate == nullptr && dw_up == nullptr && dw_down == nullptr) {
      return CCV_OK;
    }
    if (w_gate == nullptr || w_up == nullptr || w_down == nullptr ||
        (rows > 0 && (dy == nullptr || x == nullptr || saved == nullptr))) {
      return invalid("null tensor pointer");
    }
    if (rows > 1 && (x_row_stride < features || dy_row_stride < features)) {
      return invalid("row stride below the row length");
    }
    for (const void* p : {dy, x, w_gate, w_up, w_down, static_cast<const void*>(dx),
                          static_cast<const void*>(dw_gate), static_cast<const void*>(dw_up),
                          static_cast<const void*>(dw_down)}) {
      if (!aligned_to(p, 2)) return invalid("tensor pointers must be aligned to their element");
    }
    if ((rc = check_ffn_alignment(b.shape, x, x_row_stride, w_gate, w_up, w_down)) != CCV_OK ||
        (rc = check_in_place(dy, features, rows > 1 ? dy_row_stride : 0,
                             "dy must be 16-byte aligned")) != CCV_OK) {
      return rc;
    }
    for (const void* p : {static_cast<const void*>(dx), static_cast<const void*>(dw_gate),
                          static_cast<const void*>(dw_up)}) {
      if ((rc = check_in_place(p, features, 0, "gradients must be 16-byte aligned")) != CCV_OK) {
        return rc;
      }
    }
    if ((rc = check_in_place(dw_down, hidden, 0, "gradients must be 16-byte aligned")) != CCV_OK) {
      return rc;
    }
    if (rows > 0 && (!aligned_to(saved, 256) || saved_bytes < ffn_saved_planes(b.shape) * ffn_plane_bytes(b.shape))) {
      return set_error(CCV_ERR_WORKSPACE, "saved buffer misaligned or too small");
    }
    if ((rc = check_workspace(workspace, workspace_bytes,
                              ffn_backward_workspace_bytes(b.shape))) != CCV_OK) {
      return rc;
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if ((rc = begin_launches(st)) != CCV_OK) return rc;
    return launch_ffn_backward(b, workspace, st);
  });
}

int ccv_dropout(const void* x, int x_dtype, const void* residual, void* y, int y_dtype,
                int64_t count, double p, uint64_t seed, uint64_t offset,
                const int64_t* offset_device, ccv_stream_t stream) {
  return guarded([&]() -> int {
    if (valid_dtype(x_dtype) && valid_dtype(y_dtype) && residual == nullptr && y_dtype != x_dtype) {
      return invalid("without a residual the output has the input's type");
    }
    return run_dropout({x, residual, y, count, x_dtype, y_dtype, p, seed, offset, offset_device},
                       "a 16-bit input takes a residual of its own type or float32", stream);
  });
}

int ccv_dropout_backward(const void* dy, int y_dtype, void* dx, int x_dtype, int64_t count,
                         double p, uint64_t seed, uint64_t offset, const int64_t* offset_device,
                         ccv_stream_t stream) {
  return guarded([&]() -> int {
    return run_dropout({dy, nullptr, dx, count, y_dtype, x_dtype, p, seed, offset, offset_device},
                       "the gradient of a 16-bit input is of its own type or float32", stream);
  });
}

}  // extern "C"
