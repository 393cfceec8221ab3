// Gated feed-forward block, forward and backward, in 16-bit types with fp32
// sums:
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g),
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// with x [M, D], Wg and Wu [F, D], Wd [D, F].  g, u, h, dg and du are rounded
// to the operands' type once each: they are operands of the next product,
// whose inputs the tensor cores take in 16 bits.
#include "ccv_internal.h"
#include "ccv_ptx.cuh"
#include "ccv_tokens.cuh"

namespace ccv {

namespace {

__device__ __forceinline__ float act_value(int act, float g) {
  if (act == CCV_ACTIVATION_SILU) return g / (1.f + expf(-g));
  return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
}

// act(g) and act'(g).
__device__ __forceinline__ float act_slope(int act, float g, float& value) {
  if (act == CCV_ACTIVATION_SILU) {
    const float s = 1.f / (1.f + expf(-g));
    value = g * s;
    return s * (1.f + g * (1.f - s));
  }
  const float c = 0.5f * (1.f + erff(g * 0.70710678118654752f));
  value = g * c;
  return c + g * 0.39894228040143268f * expf(-0.5f * g * g);
}

// Element (i, k) of an operand at base[i * si + k * sk].
struct Operand {
  const void* base = nullptr;
  int64_t si = 0, sk = 0;
};

enum Mode { kPlain, kGate, kGrad };

struct GemmArgs {
  Operand a[2], b[2];  // kPlain: sum over both pairs (second optional); kGate: b[0] gate, b[1] up
  int64_t m = 0, n = 0, k = 0;
  void* out[3] = {};   // kPlain: C; kGate: h, g, u (g, u optional); kGrad: dg, du
  const void* in[2] = {};  // kGrad: g, u
  int64_t ldo = 0, ldi = 0;
  int act = 0;
};

constexpr int kT = 64, kTk = 16;

// 64 x 64 output tile per block, 4 x 4 per thread, fp32 multiply-adds.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) ffn_gemm_simple(const GemmArgs p) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  __shared__ float sa[kTk][kT + 1], sb[2][kTk][kT + 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kT;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kT;
  float acc[2][4][4] = {};
  const int pairs = MODE == kPlain && p.a[1].base != nullptr ? 2 : 1;
  for (int pr = 0; pr < pairs; ++pr) {
    const T* a = static_cast<const T*>(p.a[pr].base);
    for (int64_t k0 = 0; k0 < p.k; k0 += kTk) {
      for (int e = threadIdx.x; e < kT * kTk; e += 256) {
        const int i = p.a[pr].sk == 1 ? e / kTk : e % kT;
        const int k = p.a[pr].sk == 1 ? e % kTk : e / kT;
        const bool in = m0 + i < p.m && k0 + k < p.k;
        sa[k][i] = in ? to_f32(a[(m0 + i) * p.a[pr].si + (k0 + k) * p.a[pr].sk]) : 0.f;
      }
      for (int q = 0; q < (MODE == kGate ? 2 : 1); ++q) {
        const Operand& ob = MODE == kGate ? p.b[q] : p.b[pr];
        const T* b = static_cast<const T*>(ob.base);
        for (int e = threadIdx.x; e < kT * kTk; e += 256) {
          const int i = ob.sk == 1 ? e / kTk : e % kT;
          const int k = ob.sk == 1 ? e % kTk : e / kT;
          const bool in = n0 + i < p.n && k0 + k < p.k;
          sb[q][k][i] = in ? to_f32(b[(n0 + i) * ob.si + (k0 + k) * ob.sk]) : 0.f;
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kTk; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[0][i][j] += sa[k][ty * 4 + i] * sb[0][k][tx + 16 * j];
            if (MODE == kGate) acc[1][i][j] += sa[k][ty * 4 + i] * sb[1][k][tx + 16 * j];
          }
        }
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
      if (m >= p.m || n >= p.n) continue;
      const int64_t o = m * p.ldo + n;
      if (MODE == kPlain) {
        static_cast<T*>(p.out[0])[o] = from_f32<T>(acc[0][i][j]);
      } else if (MODE == kGate) {
        const float g = acc[0][i][j], u = acc[1][i][j];
        static_cast<T*>(p.out[0])[o] = from_f32<T>(act_value(p.act, g) * u);
        if (p.out[1] != nullptr) {
          static_cast<T*>(p.out[1])[o] = from_f32<T>(g);
          static_cast<T*>(p.out[2])[o] = from_f32<T>(u);
        }
      } else {
        const float g = to_f32(static_cast<const T*>(p.in[0])[m * p.ldi + n]);
        const float u = to_f32(static_cast<const T*>(p.in[1])[m * p.ldi + n]);
        float value;
        const float slope = act_slope(p.act, g, value);
        static_cast<T*>(p.out[0])[o] = from_f32<T>(acc[0][i][j] * u * slope);
        static_cast<T*>(p.out[1])[o] = from_f32<T>(acc[0][i][j] * value);
      }
    }
  }
}

template <int MODE>
int launch_gemm(const GemmArgs& a, int dtype, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((a.n + kT - 1) / kT),
                  static_cast<unsigned>((a.m + kT - 1) / kT));
  return launched(
      dtype == CCV_DTYPE_BF16
          ? launch_kernel(ffn_gemm_simple<__nv_bfloat16, MODE>, grid, dim3(256), 0, stream, 1, a)
          : launch_kernel(ffn_gemm_simple<__half, MODE>, grid, dim3(256), 0, stream, 1, a),
      "gated feed-forward product");
}

int64_t padded(int64_t n) { return (n + 7) / 8 * 8; }

}  // namespace

size_t ffn_plane_bytes(const FfnShape& s) {
  return static_cast<size_t>(s.rows) * padded(s.hidden) * 2;
}

size_t ffn_forward_workspace_bytes(const FfnShape& s) { return ffn_plane_bytes(s); }
size_t ffn_backward_workspace_bytes(const FfnShape& s) { return 2 * ffn_plane_bytes(s); }

int launch_ffn_forward(const FfnForward& f, void* ws, cudaStream_t stream) {
  const FfnShape& s = f.shape;
  if (s.rows == 0) return CCV_OK;
  const int64_t fp = padded(s.hidden);
  char* saved = static_cast<char*>(f.saved);
  const size_t plane = ffn_plane_bytes(s);
  GemmArgs a;
  a.a[0] = {f.x, f.x_stride, 1};
  a.b[0] = {f.w_gate, s.features, 1};
  a.b[1] = {f.w_up, s.features, 1};
  a.m = s.rows;
  a.n = s.hidden;
  a.k = s.features;
  a.act = s.activation;
  a.ldo = fp;
  a.out[0] = saved != nullptr ? saved : ws;
  if (saved != nullptr) {
    a.out[1] = saved + plane;
    a.out[2] = saved + 2 * plane;
  }
  int rc = launch_gemm<kGate>(a, s.dtype, stream);
  if (rc != CCV_OK) return rc;
  GemmArgs d;
  d.a[0] = {a.out[0], fp, 1};
  d.b[0] = {f.w_down, s.hidden, 1};
  d.m = s.rows;
  d.n = s.features;
  d.k = s.hidden;
  d.out[0] = f.y;
  d.ldo = s.features;
  return launch_gemm<kPlain>(d, s.dtype, stream);
}

int launch_ffn_backward(const FfnBackward& b, void* ws, cudaStream_t stream) {
  const FfnShape& s = b.shape;
  const int64_t fp = padded(s.hidden);
  const size_t plane = ffn_plane_bytes(s);
  const char* saved = static_cast<const char*>(b.saved);
  char* dg = static_cast<char*>(ws);
  char* du = dg + plane;
  int rc = CCV_OK;
  if (s.rows > 0 && (b.dx != nullptr || b.dw_gate != nullptr || b.dw_up != nullptr)) {
    GemmArgs a;
    a.a[0] = {b.dy, b.dy_stride, 1};
    a.b[0] = {b.w_down, 1, s.hidden};
    a.m = s.rows;
    a.n = s.hidden;
    a.k = s.features;
    a.in[0] = saved + plane;
    a.in[1] = saved + 2 * plane;
    a.ldi = fp;
    a.out[0] = dg;
    a.out[1] = du;
    a.ldo = fp;
    a.act = s.activation;
    if ((rc = launch_gemm<kGrad>(a, s.dtype, stream)) != CCV_OK) return rc;
  }
  if (s.rows > 0 && b.dx != nullptr) {
    GemmArgs a;
    a.a[0] = {dg, fp, 1};
    a.a[1] = {du, fp, 1};
    a.b[0] = {b.w_gate, 1, s.features};
    a.b[1] = {b.w_up, 1, s.features};
    a.m = s.rows;
    a.n = s.features;
    a.k = s.hidden;
    a.out[0] = b.dx;
    a.ldo = s.features;
    if ((rc = launch_gemm<kPlain>(a, s.dtype, stream)) != CCV_OK) return rc;
  }
  const struct {
    void* out;
    Operand a, b;
    int64_t m, n;
  } grads[3] = {
      {b.dw_gate, {dg, 1, fp}, {b.x, 1, b.x_stride}, s.hidden, s.features},
      {b.dw_up, {du, 1, fp}, {b.x, 1, b.x_stride}, s.hidden, s.features},
      {b.dw_down, {b.dy, 1, b.dy_stride}, {saved, 1, fp}, s.features, s.hidden},
  };
  for (const auto& g : grads) {
    if (g.out == nullptr) continue;
    GemmArgs a;
    a.a[0] = g.a;
    a.b[0] = g.b;
    a.m = g.m;
    a.n = g.n;
    a.k = s.rows;
    a.out[0] = g.out;
    a.ldo = g.n;
    if ((rc = launch_gemm<kPlain>(a, s.dtype, stream)) != CCV_OK) return rc;
  }
  return rc;
}

}  // namespace ccv
