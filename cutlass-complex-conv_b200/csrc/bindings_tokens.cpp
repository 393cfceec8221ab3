// Token operators of the extension `complex_conv2d._C`: checks of torch
// tensors, outputs and scratch from the caching allocator, the current
// stream, and the calls into the C ABI (include/ccv_b200.h).
#include "bindings_tokens.h"

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <string>
#include <tuple>

#include "ccv_b200.h"

namespace {

using OptTensor = c10::optional<torch::Tensor>;

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == CCV_OK, what, " failed (status ", rc, "): ", ccv_last_error_message());
}

ccv_stream_t current_stream() {
  return reinterpret_cast<ccv_stream_t>(at::cuda::getCurrentCUDAStream().stream());
}

int dtype_code(at::ScalarType t, const char* name) {
  if (t == at::kFloat) return CCV_DTYPE_F32;
  if (t == at::kBFloat16) return CCV_DTYPE_BF16;
  TORCH_CHECK_TYPE(t == at::kHalf, name, " must be float32, bfloat16 or float16, got ", t);
  return CCV_DTYPE_F16;
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// A tensor [..., features] as rows of adjacent features: in place when its
// leading dimensions collapse to one row stride, else a contiguous copy.
struct Rows {
  torch::Tensor t;
  int64_t rows = 0, features = 0, stride = 0;
};

Rows as_rows(const torch::Tensor& t) {
  Rows r;
  r.features = t.size(-1);
  r.rows = r.features > 0 ? t.numel() / r.features : 0;
  if (t.is_contiguous()) {
    r.t = t;
    r.stride = r.features;
    return r;
  }
  bool in_place = t.stride(-1) == 1 || r.features == 1;
  int64_t inner = -1;  // row stride of the dimensions seen so far
  int64_t extent = 1;
  for (int64_t d = t.dim() - 2; d >= 0 && in_place; --d) {
    if (t.size(d) == 1) continue;
    if (inner < 0) {
      inner = t.stride(d);
    } else {
      in_place = t.stride(d) == inner * extent;
    }
    extent *= t.size(d);
  }
  if (in_place) {
    r.t = t;
    r.stride = inner < 0 ? r.features : inner;
  } else {
    r.t = t.contiguous();
    r.stride = r.features;
  }
  return r;
}

void check_cuda(const torch::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
}

void check_like(const torch::Tensor& t, const torch::Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on the input's device");
}

// Uninitialised memory from the caching allocator, without the dispatcher's
// part of torch::empty (about half a microsecond of a call that takes five).
torch::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

torch::Tensor scratch(size_t bytes, const torch::Tensor& like) {
  return fresh({static_cast<int64_t>(bytes)}, torch::kUInt8, like);
}

void* ptr(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void check_norm_vector(const torch::Tensor& w, const torch::Tensor& x, const char* name) {
  check_like(w, x, name);
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(-1), name,
                    " must have one element per feature");
  TORCH_CHECK_TYPE(w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type(), name,
                   " must be float32 or of the input's type");
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> layer_norm_forward(
    torch::Tensor x, OptTensor weight, OptTensor bias, double eps,
    c10::optional<at::ScalarType> out_dtype, bool stats) {
  check_cuda(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must have at least one feature");
  const int xt = dtype_code(x.scalar_type(), "x");
  const at::ScalarType out = out_dtype.value_or(x.scalar_type());
  const int yt = dtype_code(out, "out_dtype");
  TORCH_CHECK_TYPE(xt == CCV_DTYPE_F32 || yt == CCV_DTYPE_F32 || yt == xt,
                   "a 16-bit input gives an output of its own type or float32");
  TORCH_CHECK_VALUE(eps >= 0.0, "eps must be non-negative");
  torch::Tensor w, b;
  int wt = CCV_DTYPE_F32;
  if (given(weight)) {
    check_norm_vector(*weight, x, "weight");
    w = weight->contiguous();
    wt = dtype_code(w.scalar_type(), "weight");
  }
  if (given(bias)) {
    check_norm_vector(*bias, x, "bias");
    b = bias->contiguous();
    TORCH_CHECK_TYPE(!w.defined() || w.scalar_type() == b.scalar_type(),
                     "weight and bias must have one type");
    wt = dtype_code(b.scalar_type(), "bias");
  }
  c10::cuda::CUDAGuard guard(x.device());
  const Rows r = as_rows(x);
  auto y = fresh(x.sizes(), out, x);
  torch::Tensor mean, rstd;
  if (stats) {
    const auto shape = x.sizes().slice(0, x.dim() - 1);
    mean = fresh(shape, torch::kFloat, x);
    rstd = fresh(shape, torch::kFloat, x);
  }
  check_rc(ccv_layer_norm_forward(r.t.data_ptr(), xt, r.stride, ptr(w), ptr(b), wt,
                                  static_cast<float>(eps), y.data_ptr(), yt,
                                  static_cast<float*>(ptr(mean)), static_cast<float*>(ptr(rstd)),
                                  r.rows, r.features, current_stream()),
           "ccv_layer_norm_forward");
  return {y, mean, rstd};
}

// needs: which of dx, dweight, dbias to compute.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> layer_norm_backward(
    torch::Tensor dy, torch::Tensor x, torch::Tensor mean, torch::Tensor rstd, OptTensor weight,
    c10::optional<at::ScalarType> weight_dtype, bool need_dx, bool need_dweight, bool need_dbias) {
  check_cuda(x, "x");
  check_like(dy, x, "dy");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must have at least one feature");
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "dy must have the input's shape");
  const int xt = dtype_code(x.scalar_type(), "x");
  const int yt = dtype_code(dy.scalar_type(), "dy");
  TORCH_CHECK_TYPE(xt == CCV_DTYPE_F32 || yt == CCV_DTYPE_F32 || yt == xt,
                   "dy must be float32 or of the 16-bit input's type");
  const Rows rx = as_rows(x), rdy = as_rows(dy);
  for (const auto* t : {&mean, &rstd}) {
    check_like(*t, x, "mean and rstd");
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, "mean and rstd must be float32");
    TORCH_CHECK_VALUE(t->numel() == rx.rows, "mean and rstd must have one element per row");
  }
  mean = mean.contiguous();
  rstd = rstd.contiguous();
  torch::Tensor w;
  at::ScalarType wtype = weight_dtype.value_or(at::kFloat);
  if (given(weight)) {
    check_norm_vector(*weight, x, "weight");
    w = weight->contiguous();
    wtype = w.scalar_type();
  }
  const int wt = dtype_code(wtype, "weight");
  c10::cuda::CUDAGuard guard(x.device());
  torch::Tensor dx, dw, db;
  if (need_dx) dx = fresh(x.sizes(), x.scalar_type(), x);
  if (need_dweight) dw = fresh({rx.features}, wtype, x);
  if (need_dbias) db = fresh({rx.features}, wtype, x);
  const size_t bytes = ccv_layer_norm_backward_workspace_bytes(rx.rows, rx.features);
  auto ws = scratch(bytes, x);
  check_rc(ccv_layer_norm_backward(rdy.t.data_ptr(), yt, rdy.stride, rx.t.data_ptr(), xt, rx.stride,
                                   mean.data_ptr<float>(), rstd.data_ptr<float>(), ptr(w), wt,
                                   ptr(dx), ptr(dw), ptr(db), rx.rows, rx.features, ptr(ws), bytes,
                                   current_stream()),
           "ccv_layer_norm_backward");
  return {dx, dw, db};
}

// Rows that TMA can read in place where their length allows it at all.
Rows as_tma_rows(const torch::Tensor& t) {
  Rows r = as_rows(t);
  const bool overlap = r.rows > 1 && r.stride < r.features;  // expanded rows
  if (overlap || (r.features % 8 == 0 && (reinterpret_cast<uintptr_t>(r.t.data_ptr()) % 16 != 0 ||
                                          (r.rows > 1 && r.stride % 8 != 0)))) {
    r.t = t.clone(at::MemoryFormat::Contiguous);
    r.stride = r.features;
  }
  if (r.rows <= 1) r.stride = r.features;
  return r;
}

torch::Tensor aligned_weight(const torch::Tensor& w) {
  return as_tma_rows(w.contiguous()).t;
}

struct FfnWeights {
  torch::Tensor gate, up, down;
  int64_t hidden = 0;
};

FfnWeights check_ffn(const torch::Tensor& x, const torch::Tensor& w_gate,
                     const torch::Tensor& w_up, const torch::Tensor& w_down) {
  check_cuda(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must have at least one feature");
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
                   "the gated feed-forward block takes bfloat16 or float16, got ",
                   x.scalar_type());
  const int64_t d = x.size(-1);
  TORCH_CHECK_VALUE(w_gate.dim() == 2 && w_gate.size(1) == d && w_gate.size(0) > 0,
                    "w_gate must be [hidden, features]");
  const int64_t f = w_gate.size(0);
  TORCH_CHECK_VALUE(w_up.dim() == 2 && w_up.size(0) == f && w_up.size(1) == d,
                    "w_up must be [hidden, features]");
  TORCH_CHECK_VALUE(w_down.dim() == 2 && w_down.size(0) == d && w_down.size(1) == f,
                    "w_down must be [features, hidden]");
  for (const auto* w : {&w_gate, &w_up, &w_down}) {
    check_like(*w, x, "weights");
    TORCH_CHECK_TYPE(w->scalar_type() == x.scalar_type(), "weights must be of the input's type");
  }
  return {aligned_weight(w_gate), aligned_weight(w_up), aligned_weight(w_down), f};
}

// Columns of a plane of the saved buffer (rows of whole 16-byte units).
int64_t saved_width(int64_t hidden) { return (hidden + 7) / 8 * 8; }

// Its planes: what the library asks for, by the size of one.
int64_t saved_planes(int64_t rows, int64_t features, int64_t hidden) {
  rows = rows > 0 ? rows : 1;
  return static_cast<int64_t>(ccv_gated_ffn_saved_bytes(rows, features, hidden)) /
         (2 * rows * saved_width(hidden));
}

int activation_code(const std::string& name) {
  if (name == "silu") return CCV_ACTIVATION_SILU;
  TORCH_CHECK_VALUE(name == "gelu", "activation must be 'silu' or 'gelu', got '", name, "'");
  return CCV_ACTIVATION_GELU;
}

std::tuple<torch::Tensor, torch::Tensor> gated_ffn_forward(torch::Tensor x, torch::Tensor w_gate,
                                                           torch::Tensor w_up,
                                                           torch::Tensor w_down,
                                                           const std::string& activation,
                                                           bool save) {
  const int act = activation_code(activation);
  check_cuda(x, "x");
  c10::cuda::CUDAGuard guard(x.device());
  const FfnWeights w = check_ffn(x, w_gate, w_up, w_down);
  const Rows r = as_tma_rows(x);
  auto y = fresh(x.sizes(), x.scalar_type(), x);
  torch::Tensor saved;
  size_t saved_bytes = 0;
  if (save) {
    saved_bytes = ccv_gated_ffn_saved_bytes(r.rows, r.features, w.hidden);
    saved = fresh({saved_planes(r.rows, r.features, w.hidden), r.rows, saved_width(w.hidden)},
                  x.scalar_type(), x);
  }
  const size_t bytes = ccv_gated_ffn_forward_workspace_bytes(r.rows, r.features, w.hidden, save);
  auto ws = scratch(bytes, x);
  check_rc(ccv_gated_ffn_forward(r.t.data_ptr(), r.stride, w.gate.data_ptr(), w.up.data_ptr(),
                                 w.down.data_ptr(), y.data_ptr(),
                                 dtype_code(x.scalar_type(), "x"), act, r.rows, r.features,
                                 w.hidden, ptr(saved), saved_bytes, ptr(ws), bytes,
                                 current_stream()),
           "ccv_gated_ffn_forward");
  return {y, saved};
}

// needs: which of dx, dw_gate, dw_up, dw_down to compute.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> gated_ffn_backward(
    torch::Tensor dy, torch::Tensor saved, torch::Tensor x, torch::Tensor w_gate,
    torch::Tensor w_up, torch::Tensor w_down, const std::string& activation, bool need_dx,
    bool need_dgate, bool need_dup, bool need_ddown) {
  const int act = activation_code(activation);
  check_cuda(x, "x");
  c10::cuda::CUDAGuard guard(x.device());
  const FfnWeights w = check_ffn(x, w_gate, w_up, w_down);
  check_like(dy, x, "dy");
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "dy must have the input's shape");
  TORCH_CHECK_TYPE(dy.scalar_type() == x.scalar_type(), "dy must be of the input's type");
  check_like(saved, x, "saved");
  const Rows rx = as_tma_rows(x), rdy = as_tma_rows(dy);
  TORCH_CHECK_VALUE(saved.scalar_type() == x.scalar_type() && saved.is_contiguous() &&
                        saved.dim() == 3 && saved.size(0) == saved_planes(rx.rows, rx.features, w.hidden) && saved.size(1) == rx.rows &&
                        saved.size(2) == saved_width(w.hidden),
                    "saved must be what the forward call returned for these shapes");
  torch::Tensor dx, dg, du, dd;
  if (need_dx) dx = fresh(x.sizes(), x.scalar_type(), x);
  if (need_dgate) dg = fresh(w.gate.sizes(), x.scalar_type(), x);
  if (need_dup) du = fresh(w.up.sizes(), x.scalar_type(), x);
  if (need_ddown) dd = fresh(w.down.sizes(), x.scalar_type(), x);
  const size_t bytes = ccv_gated_ffn_backward_workspace_bytes(rx.rows, rx.features, w.hidden);
  auto ws = scratch(bytes, x);
  check_rc(ccv_gated_ffn_backward(rdy.t.data_ptr(), rdy.stride, rx.t.data_ptr(), rx.stride,
                                  w.gate.data_ptr(), w.up.data_ptr(), w.down.data_ptr(),
                                  saved.data_ptr(), static_cast<size_t>(saved.numel()) * 2, ptr(dx),
                                  ptr(dg), ptr(du), ptr(dd), dtype_code(x.scalar_type(), "x"), act,
                                  rx.rows, rx.features, w.hidden, ptr(ws), bytes,
                                  current_stream()),
           "ccv_gated_ffn_backward");
  return {dx, dg, du, dd};
}

const int64_t* check_offset(const OptTensor& offset, const torch::Tensor& x) {
  if (!given(offset)) return nullptr;
  check_like(*offset, x, "offset");
  TORCH_CHECK_TYPE(offset->scalar_type() == at::kLong, "offset must be an int64 tensor");
  TORCH_CHECK_VALUE(offset->numel() == 1, "offset must have one element");
  return offset->data_ptr<int64_t>();
}

torch::Tensor dropout(torch::Tensor x, double p, uint64_t seed, uint64_t offset,
                      OptTensor offset_device, OptTensor residual) {
  check_cuda(x, "x");
  const int xt = dtype_code(x.scalar_type(), "x");
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be between 0 and 1, got ", p);
  at::ScalarType out = x.scalar_type();
  torch::Tensor r;
  if (given(residual)) {
    check_like(*residual, x, "residual");
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "residual must have the input's shape");
    out = residual->scalar_type();
    r = residual->contiguous();
  }
  const int yt = dtype_code(out, "residual");
  TORCH_CHECK_TYPE(xt == CCV_DTYPE_F32 || yt == CCV_DTYPE_F32 || yt == xt,
                   "residual must be float32 or of the 16-bit input's type");
  const int64_t* od = check_offset(offset_device, x);
  c10::cuda::CUDAGuard guard(x.device());
  auto xc = x.contiguous();
  auto y = fresh(x.sizes(), out, x);
  check_rc(ccv_dropout(xc.data_ptr(), xt, ptr(r), y.data_ptr(), yt, x.numel(), p, seed, offset, od,
                       current_stream()),
           "ccv_dropout");
  return y;
}

torch::Tensor dropout_backward(torch::Tensor dy, double p, uint64_t seed, uint64_t offset,
                               OptTensor offset_device, at::ScalarType x_dtype) {
  check_cuda(dy, "dy");
  const int yt = dtype_code(dy.scalar_type(), "dy");
  const int xt = dtype_code(x_dtype, "x_dtype");
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be between 0 and 1, got ", p);
  TORCH_CHECK_TYPE(xt == CCV_DTYPE_F32 || yt == CCV_DTYPE_F32 || yt == xt,
                   "dy must be float32 or of the 16-bit input's type");
  const int64_t* od = check_offset(offset_device, dy);
  c10::cuda::CUDAGuard guard(dy.device());
  auto g = dy.contiguous();
  auto dx = fresh(dy.sizes(), x_dtype, dy);
  check_rc(ccv_dropout_backward(g.data_ptr(), yt, dx.data_ptr(), xt, dy.numel(), p, seed, offset, od,
                                current_stream()),
           "ccv_dropout_backward");
  return dx;
}

}  // namespace

void register_token_operators(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("layer_norm_forward", &layer_norm_forward, "layer norm -> (y, mean, rstd)", py::arg("x"),
        py::arg("weight"), py::arg("bias"), py::arg("eps"), py::arg("out_dtype"),
        py::arg("stats"));
  m.def("layer_norm_backward", &layer_norm_backward, "-> (dx, dweight, dbias)", py::arg("dy"),
        py::arg("x"), py::arg("mean"), py::arg("rstd"), py::arg("weight"),
        py::arg("weight_dtype"), py::arg("need_dx"), py::arg("need_dweight"),
        py::arg("need_dbias"));
  m.def("gated_ffn_forward", &gated_ffn_forward, "gated feed-forward block -> (y, saved)",
        py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"),
        py::arg("activation"), py::arg("save"));
  m.def("gated_ffn_backward", &gated_ffn_backward, "-> (dx, dw_gate, dw_up, dw_down)",
        py::arg("dy"), py::arg("saved"), py::arg("x"), py::arg("w_gate"), py::arg("w_up"),
        py::arg("w_down"), py::arg("activation"), py::arg("need_dx"), py::arg("need_dgate"),
        py::arg("need_dup"), py::arg("need_ddown"));
  m.def("dropout", &dropout, "counter-based dropout", py::arg("x"), py::arg("p"),
        py::arg("seed"), py::arg("offset"), py::arg("offset_device"), py::arg("residual"));
  m.def("dropout_backward", &dropout_backward, "-> dx", py::arg("dy"), py::arg("p"),
        py::arg("seed"), py::arg("offset"), py::arg("offset_device"), py::arg("x_dtype"));
}
