// Gated feed-forward block, forward and backward, in 16-bit types with fp32
// sums:
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g),
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// with x [M, D], Wg and Wu [F, D], Wd [D, F].  h, dg and du are rounded to the
// operands' type once each: they are operands of the next product, whose
// inputs the tensor cores take in 16 bits.  g and u are computed again in the
// backward pass, or (many features) kept for it to 24 bits.
//
// Forward: GATE, PLAIN.  Backward: GRAD or REGRAD, PLAIN over two segments (dx), PLAIN
// over three problems in one launch (the weight gradients).  This file plans
// the tiles, builds the tensor maps and launches ccv_ffn_gemm.cuh's kernel.
//
// TMA wants row lengths that are multiples of 16 bytes: where D or F is not
// a multiple of 8, the matrices with such rows are copied to padded rows in
// the workspace first, and results come back through one.
#include <algorithm>
#include <mutex>

#include "ccv_ffn_gemm.cuh"
#include "ccv_ffn_rows.cuh"
#include "ccv_internal.h"
#include "ccv_ptx.cuh"
#include "ccv_tokens.cuh"

namespace ccv {

namespace {

using ffn::GemmParams;

int64_t padded(int64_t n) { return (n + 7) / 8 * 8; }

size_t align256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }

// Carves a workspace; with a null base it only adds up the size.
struct Carver {
  char* base;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = base != nullptr ? base + used : nullptr;
    used += align256(bytes);
    return p;
  }
};

// ------------------------------------------------------------ small kernels
// Matrices of 16-bit elements from one row pitch to another, all in one
// launch (blockIdx.y is the matrix): a call with odd sizes copies up to five.
struct RowCopy {
  const uint16_t* src;
  uint16_t* dst;
  int64_t src_pitch, dst_pitch, rows;
  int cols;
};
struct RowCopies {
  RowCopy m[5];
  int count = 0;
  void add(const void* src, int64_t src_pitch, void* dst, int64_t dst_pitch, int64_t rows,
           int64_t cols) {
    m[count++] = {static_cast<const uint16_t*>(src), static_cast<uint16_t*>(dst), src_pitch,
                  dst_pitch, rows, static_cast<int>(cols)};
  }
};

constexpr int kCopyAhead = 16;  // loads in flight per lane

__global__ void __launch_bounds__(256) ffn_copy_rows(const RowCopies c) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const RowCopy& m = c.m[blockIdx.y];
  const int lane = threadIdx.x & 31;
  for (int64_t r = blockIdx.x * 8 + (threadIdx.x >> 5); r < m.rows; r += gridDim.x * 8) {
    const uint16_t* src = m.src + r * m.src_pitch;
    uint16_t* dst = m.dst + r * m.dst_pitch;
    for (int k0 = lane; k0 < m.cols; k0 += 32 * kCopyAhead) {
      uint16_t v[kCopyAhead];
#pragma unroll
      for (int i = 0; i < kCopyAhead; ++i) {
        if (k0 + 32 * i < m.cols) v[i] = src[k0 + 32 * i];
      }
#pragma unroll
      for (int i = 0; i < kCopyAhead; ++i) {
        if (k0 + 32 * i < m.cols) dst[k0 + 32 * i] = v[i];
      }
    }
  }
}

int copy_rows(const RowCopies& c, cudaStream_t stream) {
  if (c.count == 0) return CCV_OK;
  int64_t most = 1;
  for (int i = 0; i < c.count; ++i) most = std::max(most, c.m[i].rows);
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((most + 7) / 8, device_sm_count() * 8));
  return launched(
      launch_kernel(ffn_copy_rows, dim3(blocks, c.count), dim3(256), 0, stream, 1, c), "row copy");
}

struct SplitSum {
  const float* partial;  // [split tile][split][256][bn]
  ffn::Tiles tiles[ffn::kMaxProblems];
  void* out[ffn::kMaxProblems];
  int64_t ldo[ffn::kMaxProblems];
  int problems, whole, splits, bn;
};

// The split tiles' results: their parts added in order, four columns per
// thread; blockIdx.y is the tile.
template <typename T>
__global__ void __launch_bounds__(256) ffn_split_sum(const SplitSum p) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  int problem, tm, tn;
  ffn::locate(p.tiles, p.problems, p.whole + static_cast<int>(blockIdx.y), problem, tm, tn);
  const int quads = p.bn / 4;
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int r = i / quads, c = (i - r * quads) * 4;
  const int64_t row = static_cast<int64_t>(tm) * 256 + r, col = static_cast<int64_t>(tn) * p.bn + c;
  const ffn::Tiles& t = p.tiles[problem];
  if (row >= t.m || col >= t.n) return;
  const int64_t part = 256LL * p.bn;
  const float* src = p.partial + blockIdx.y * part * p.splits + static_cast<int64_t>(r) * p.bn + c;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < p.splits; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(src + k * part);
    a.x += v.x;
    a.y += v.y;
    a.z += v.z;
    a.w += v.w;
  }
  T* o = static_cast<T*>(p.out[problem]) + row * p.ldo[problem] + col;
  const float f[4] = {a.x, a.y, a.z, a.w};
  if (p.ldo[problem] % 4 == 0 && (reinterpret_cast<uintptr_t>(o) & 7) == 0 && col + 4 <= t.n) {
    store_vec<T, 4>(o, f);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (col + j < t.n) o[j] = from_f32<T>(f[j]);
  }
}

// ------------------------------------------------------------ few rows
// Up to this many rows the block streams its weights through mma.sync.  Against
// the tcgen05 tiles, bf16 SiLU, calls back to back on B200 (us):
//            256 x 1024    512 x 2048    1024 x 4096   2048 x 8192
//    1 row   4.7 / 13.6    5.5 / 14.7    10.2 / 25.0   26.3 / 43.1
//    8 rows  4.7 / 13.6    5.7 / 14.4    12.0 / 21.3   30.4 / 38.2
//   16 rows  6.3 / 13.6    7.8 / 14.4    15.8 / 21.3   39.4 / 38.0
//   17 rows  7.4 / 13.6    9.1 / 14.4    20.4 / 21.4   46.1 / 38.2
//   32 rows  8.8 / 13.7   11.1 / 14.5    26.2 / 21.5   60.1 / 35.8
// (17 and more: instances for 24 and 32 rows, which only narrow blocks would
// gain by and which are not built.)
constexpr int64_t kFewRows = 16;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, int NT>
int launch_rows(const FfnForward& f, void* h, void* const (&planes)[3], cudaStream_t stream) {
  const FfnShape& s = f.shape;
  const int64_t sms = device_sm_count(), fp = padded(s.hidden);
  ffn::RowsParams p = {};
  p.x = static_cast<const uint16_t*>(f.x);
  p.x_stride = f.x_stride;
  p.w0 = static_cast<const uint16_t*>(f.w_gate);
  p.w1 = static_cast<const uint16_t*>(f.w_up);
  p.out = static_cast<uint16_t*>(h);
  p.g = static_cast<uint16_t*>(planes[0]);
  p.u = static_cast<uint16_t*>(planes[1]);
  p.next = static_cast<uint16_t*>(planes[2]);
  p.out_stride = fp;
  p.rows = static_cast<int>(s.rows);
  p.k = static_cast<int>(s.features);
  p.outputs = static_cast<int>(s.hidden);
  p.act = s.activation;
  // Groups of 8 outputs per block: as many as leave four blocks per SM.
  const int64_t groups = (s.hidden + 7) / 8;
  p.blocks_per_cta = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, groups / (4 * sms))));
  const bool vec = s.features % 8 == 0 && aligned16(f.x) && f.x_stride % 8 == 0 &&
                   aligned16(f.w_gate) && aligned16(f.w_up);
  const dim3 gate_grid(static_cast<unsigned>((groups + p.blocks_per_cta - 1) / p.blocks_per_cta));
  int rc = launched(
      vec ? launch_kernel(ffn::ffn_rows_gate<T, NT, true>, gate_grid, dim3(ffn::kRowsThreads), 0,
                          stream, 1, p)
          : launch_kernel(ffn::ffn_rows_gate<T, NT, false>, gate_grid, dim3(ffn::kRowsThreads), 0,
                          stream, 1, p),
      "gated feed-forward gate");
  if (rc != CCV_OK) return rc;
  ffn::RowsParams d = {};
  d.x = static_cast<const uint16_t*>(h);
  d.x_stride = fp;
  d.w0 = static_cast<const uint16_t*>(f.w_down);
  d.out = static_cast<uint16_t*>(f.y);
  d.out_stride = s.features;
  d.rows = p.rows;
  d.k = p.outputs;
  d.outputs = p.k;
  // Blocks per cluster: enough for two blocks per SM, while each warp keeps
  // two chunks of the reduction.
  const int64_t tiles = (s.features + 15) / 16;
  int cluster = 1;
  while (cluster < 8 && tiles * cluster < 2 * sms &&
         s.hidden >= static_cast<int64_t>(2 * cluster) * ffn::kRowsWarps * 2 * ffn::kChunk) {
    cluster *= 2;
  }
  const dim3 down_grid(static_cast<unsigned>(tiles * cluster));
  const bool vec_w = s.hidden % 8 == 0 && aligned16(f.w_down);
  return launched(
      vec_w ? launch_kernel(ffn::ffn_rows_down<T, NT, true>, down_grid, dim3(ffn::kRowsThreads), 0,
                            stream, cluster, d)
            : launch_kernel(ffn::ffn_rows_down<T, NT, false>, down_grid, dim3(ffn::kRowsThreads), 0,
                            stream, cluster, d),
      "gated feed-forward down");
}

template <typename T>
int run_rows(const FfnForward& f, void* h, void* const (&planes)[3], cudaStream_t stream) {
  return f.shape.rows <= 8 ? launch_rows<T, 1>(f, h, planes, stream)
                           : launch_rows<T, 2>(f, h, planes, stream);
}

// Up to this many features the backward pass computes g and u again (4 D
// operations per row and hidden unit) instead of reading what the forward
// pass kept (6 bytes written and read), which also takes a quarter of the
// memory.  Both passes together, kept against computed again, bf16 SiLU:
// 25088 x 256 x 1024 182 / 155 us, 25088 x 384 x 1024 230 / 216, 12544 x 512 x
// 2048 258 / 252, 8192 x 768 x 3200 334 / 346, 8192 x 1024 x 4096 504 / 549.
// Not where there are fewer than two waves of tiles: there the doubled chain
// of K steps is what counts (600 x 360 x 704 backward 22.5 / 24.7).
constexpr int64_t kRecomputeFeatures = 512;

// ------------------------------------------------------------ planning
struct Extent {
  int64_t m, n;
};

struct Plan {
  int bn = 256;
  int64_t whole = 0;   // tiles that one unit computes
  int64_t tail = 0;    // the others, in `splits` parts each
  int splits = 1;
  size_t partial_bytes() const {
    return static_cast<size_t>(tail) * splits * 256 * bn * sizeof(float);
  }
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t tile_count(const Extent* e, int problems, int width) {
  int64_t t = 0;
  for (int i = 0; i < problems; ++i) t += ceil_div(e[i].m, 256) * ceil_div(e[i].n, width);
  return t;
}

// Tile width, and the split of the tiles past the last full wave, by an
// estimate in clocks.  A K step of a 256 x 256 tile is 512 clocks of
// multiplication; of a 256 x 128 tile it measured 0.85 times that on B200,
// not half, because the narrower tile reads as much of A from shared memory
// (128 bytes a clock is all there is).  Tiles that fill whole waves of the
// clusters are never split; the rest may be, so that the last wave is short,
// at the cost of a second launch and of the partial sums' traffic.
Plan make_plan(const Extent* e, int problems, int64_t ksteps, bool may_split, bool gate) {
  const int64_t clusters = std::max(1, device_sm_count() / 2);
  Plan best;
  double best_cost = 1e30;
  for (int bn : {256, 128}) {
    if (knobs().ffn_bn != 0 && knobs().ffn_bn != bn) continue;
    const int64_t tiles = tile_count(e, problems, gate ? bn / 2 : bn);
    const double step = bn == 256 ? 512.0 : 435.0;
    const int64_t full = tiles / clusters * clusters;
    const int64_t rest = tiles - full;
    const double base = static_cast<double>(full / clusters) * ksteps * step;
    const int most = rest > 0 && may_split ? static_cast<int>(std::min<int64_t>(64, ksteps)) : 1;
    for (int splits = 1; splits <= most; ++splits) {
      if (knobs().ffn_splits != 0 && splits != std::min(most, knobs().ffn_splits)) continue;
      double cost = base;
      if (rest > 0) {
        cost += static_cast<double>(ceil_div(rest * splits, clusters) * ceil_div(ksteps, splits)) *
                step;
      }
      if (splits > 1) cost += 5000.0 + 8.0 * rest * splits * 256 * bn / 3500.0;
      if (cost < best_cost * 0.999) {
        best_cost = cost;
        best.bn = bn;
        best.splits = splits;
        best.whole = splits > 1 ? full : tiles;
        best.tail = splits > 1 ? rest : 0;
      }
    }
  }
  return best;
}

// ------------------------------------------------------------ tensor maps
CUtensorMapDataType map_type(int dtype) {
  return dtype == CCV_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

int encode_2d(CUtensorMap* map, int dtype, const void* base, int64_t inner, int64_t outer,
              int64_t ld, int box_inner, int box_outer) {
  const uint64_t dims[2] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(outer)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld) * 2};
  const uint32_t box[2] = {static_cast<uint32_t>(box_inner), static_cast<uint32_t>(box_outer)};
  const uint32_t es[2] = {1, 1};
  return encode_tiled_typed(map, map_type(dtype), base, 2, dims, strides, box, es,
                            box_inner == 32 ? kSwizzle64 : kSwizzle128);
}

// A matrix in memory: `inner` adjacent elements per row, rows `ld` apart.
struct Matrix {
  const void* base = nullptr;
  int64_t inner = 0, outer = 0, ld = 0;
};

template <typename T, int MODE, int BN, bool A_MN, bool B_MN, int ACT>
int launch_variant(const GemmParams& prm, cudaStream_t stream) {
  using C = ffn::Config<MODE, BN>;
  auto kern = ffn::ffn_gemm_kernel<T, MODE, BN, A_MN, B_MN, ACT>;
  static std::once_flag once[64];
  static int max_clusters[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (err != cudaSuccess) return;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(4 * device_sm_count(), 1, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmem;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess && n > 0) {
      max_clusters[dev & 63] = n;
    } else {
      cudaGetLastError();
      max_clusters[dev & 63] = device_sm_count() / 2 * C::kBlocksPerSm;
    }
  });
  if (err != cudaSuccess) return cuda_error(err, "cudaFuncSetAttribute(ffn)");
  const int clusters = std::min(prm.units, std::max(1, max_clusters[dev & 63]));
  return launched(launch_kernel(kern, dim3(2 * clusters), dim3(C::kThreads), C::kSmem, stream, 0,
                                prm),
                  "gated feed-forward product");
}

template <typename T, int MODE, bool A_MN, bool B_MN>
int launch_typed(const GemmParams& prm, int bn, int act, cudaStream_t stream) {
  constexpr int kSilu = CCV_ACTIVATION_SILU, kGelu = CCV_ACTIVATION_GELU;
  if constexpr (MODE == ffn::REGRAD) {  // of one width
    return act == kGelu ? launch_variant<T, MODE, 256, A_MN, B_MN, kGelu>(prm, stream)
                        : launch_variant<T, MODE, 256, A_MN, B_MN, kSilu>(prm, stream);
  } else {
    if constexpr (MODE != ffn::PLAIN) {
      if (act == kGelu) {
        return bn == 256 ? launch_variant<T, MODE, 256, A_MN, B_MN, kGelu>(prm, stream)
                         : launch_variant<T, MODE, 128, A_MN, B_MN, kGelu>(prm, stream);
      }
    }
    return bn == 256 ? launch_variant<T, MODE, 256, A_MN, B_MN, kSilu>(prm, stream)
                     : launch_variant<T, MODE, 128, A_MN, B_MN, kSilu>(prm, stream);
  }
}

template <int MODE, bool A_MN, bool B_MN>
int launch_product(const GemmParams& prm, int dtype, int bn, int act, cudaStream_t stream) {
  return dtype == CCV_DTYPE_BF16
             ? launch_typed<__nv_bfloat16, MODE, A_MN, B_MN>(prm, bn, act, stream)
             : launch_typed<__half, MODE, A_MN, B_MN>(prm, bn, act, stream);
}

// One launch under construction.
template <int MODE, bool A_MN, bool B_MN>
struct Product {
  GemmParams prm = {};
  Plan plan;
  SplitSum sums = {};
  int dtype, act;
  int64_t tiles = 0;
  int rc = CCV_OK;

  Product(int dtype_, const Plan& plan_, int64_t k, int act_)
      : plan(plan_), dtype(dtype_), act(act_) {
    prm.status = device_status_ptr();
    prm.problems = 1;
    prm.segments = 1;
    prm.ksteps = static_cast<int>(ceil_div(k, ffn::kStepK));
    prm.splits = plan.splits;
    prm.whole = static_cast<int>(plan.whole);
  }
  void operand_a(int i, const Matrix& x) {
    if (rc == CCV_OK) {
      rc = encode_2d(&prm.a[i], dtype, x.base, x.inner, x.outer, x.ld, 64, A_MN ? 64 : ffn::kRows);
    }
  }
  void operand_b(int i, const Matrix& x) {
    if (rc == CCV_OK) {
      rc = encode_2d(&prm.b[i], dtype, x.base, x.inner, x.outer, x.ld, 64,
                     B_MN ? 64 : plan.bn / 2);
    }
  }
  // Columns of an epilogue warp's stores.
  int out_box() const {
    return MODE == ffn::PLAIN ? 64 : 32;
  }
  void result(int i, void* base, int64_t m, int64_t n, int64_t ld) {
    if (rc == CCV_OK) rc = encode_2d(&prm.out[i], dtype, base, n, m, ld, out_box(), 32);
    sums.out[i] = base;
    sums.ldo[i] = ld;
  }
  // A plane of 16-bit words read or written beside the results.
  void plane(CUtensorMap* map, const void* base, int64_t m, int64_t n, int64_t ld) {
    if (rc == CCV_OK) rc = encode_2d(map, dtype, base, n, m, ld, out_box(), 32);
  }
  // Storage for the split tiles' parts (none without a split).
  void partials(void* base) {
    if (plan.tail == 0 || rc != CCV_OK) return;
    const uint64_t bn = static_cast<uint64_t>(plan.bn);
    const uint64_t dims[3] = {bn, 256, static_cast<uint64_t>(plan.tail * plan.splits)};
    const uint64_t strides[2] = {bn * 4, bn * 4 * 256};
    const uint32_t box[3] = {32, 32, 1};
    const uint32_t es[3] = {1, 1, 1};
    sums.partial = static_cast<const float*>(base);
    rc = encode_tiled_typed(&prm.partial, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, base, 3, dims, strides,
                            box, es, kSwizzle128);
  }
  void problem(int i, int64_t m, int64_t n) {
    ffn::Tiles& t = prm.tiles[i];
    t.m = static_cast<int>(m);
    t.n = static_cast<int>(n);
    t.tiles_m = static_cast<int>(ceil_div(m, 256));
    constexpr bool gated = MODE == ffn::GATE || MODE == ffn::REGRAD;
    t.tiles_n = static_cast<int>(ceil_div(n, gated ? plan.bn / 2 : plan.bn));
    t.first = static_cast<int>(tiles);
    t.band_inverse = static_cast<uint32_t>((1ULL << 32) / (ffn::kRasterRows * static_cast<uint64_t>(t.tiles_n)));
    tiles += static_cast<int64_t>(t.tiles_m) * t.tiles_n;
    prm.problems = i + 1;
  }
  int launch(cudaStream_t stream) {
    if (rc != CCV_OK) return rc;
    if (prm.status == nullptr) return CCV_ERR_DEVICE;
    // Fewer problems than planned for leave fewer tiles.
    prm.whole = static_cast<int>(MODE == ffn::REGRAD ? tiles : std::min<int64_t>(plan.whole, tiles));
    const int64_t tail = tiles - prm.whole;
    const int64_t units = prm.whole + tail * plan.splits;
    if (units > 0x7fffffff) return set_error(CCV_ERR_UNSUPPORTED, "tensor too large");
    prm.units = static_cast<int>(units);
    const int launched_rc = launch_product<MODE, A_MN, B_MN>(prm, dtype, plan.bn, act, stream);
    if (launched_rc != CCV_OK || tail == 0) return launched_rc;
    for (int i = 0; i < prm.problems; ++i) sums.tiles[i] = prm.tiles[i];
    sums.problems = prm.problems;
    sums.whole = prm.whole;
    sums.splits = plan.splits;
    sums.bn = plan.bn;
    const dim3 grid(static_cast<unsigned>(plan.bn / 4), static_cast<unsigned>(tail));
    return launched(
        dtype == CCV_DTYPE_BF16
            ? launch_kernel(ffn_split_sum<__nv_bfloat16>, grid, dim3(256), 0, stream, 1, sums)
            : launch_kernel(ffn_split_sum<__half>, grid, dim3(256), 0, stream, 1, sums),
        "gated feed-forward split sum");
  }
};

// A [rows][cols] operand with rows TMA can read: itself, or its padded copy.
struct Padded {
  const void* src;
  int64_t src_ld, rows, cols;
  void* copy = nullptr;  // null: src is used
  Matrix matrix() const {
    return {copy != nullptr ? copy : src, cols, rows, copy != nullptr ? padded(cols) : src_ld};
  }
  void fill(RowCopies& c) const {
    if (copy != nullptr) c.add(src, src_ld, copy, padded(cols), rows, cols);
  }
};

void* take_rows(Carver& c, int64_t rows, int64_t cols) {
  return c.take(static_cast<size_t>(rows) * padded(cols) * 2);
}

struct ForwardPlan {
  bool pad_d = false, pad_f = false;
  Plan gate, down;
  void *h = nullptr, *x = nullptr, *w_gate = nullptr, *w_up = nullptr, *w_down = nullptr,
       *y = nullptr, *partial = nullptr;
};

ForwardPlan plan_forward(const FfnShape& s, bool save, Carver& c) {
  ForwardPlan p;
  if (s.rows <= kFewRows) {
    if (!save) p.h = take_rows(c, s.rows, s.hidden);
    return p;
  }
  p.pad_d = s.features % 8 != 0;
  p.pad_f = s.hidden % 8 != 0;
  const Extent eh = {s.rows, s.hidden}, ey = {s.rows, s.features};
  p.gate = make_plan(&eh, 1, ceil_div(s.features, ffn::kStepK), false, true);
  p.down = make_plan(&ey, 1, ceil_div(s.hidden, ffn::kStepK), true, false);
  if (!save) p.h = take_rows(c, s.rows, s.hidden);
  if (p.pad_d) {
    p.x = take_rows(c, s.rows, s.features);
    p.w_gate = take_rows(c, s.hidden, s.features);
    p.w_up = take_rows(c, s.hidden, s.features);
    p.y = take_rows(c, s.rows, s.features);
  }
  if (p.pad_f) p.w_down = take_rows(c, s.features, s.hidden);
  p.partial = c.take(p.down.partial_bytes());
  return p;
}

struct BackwardPlan {
  bool pad_d, pad_f;
  Plan grad, dx, dw;
  Extent dw_extent[3];
  void *dg, *du, *dy = nullptr, *x = nullptr, *w_gate = nullptr, *w_up = nullptr,
                 *w_down = nullptr, *out_dx = nullptr, *out_dw[3] = {}, *partial = nullptr;
};

BackwardPlan plan_backward(const FfnShape& s, Carver& c) {
  BackwardPlan p;
  p.pad_d = s.features % 8 != 0;
  p.pad_f = s.hidden % 8 != 0;
  const Extent eh = {s.rows, s.hidden}, ex = {s.rows, s.features};
  p.dw_extent[0] = p.dw_extent[1] = {s.hidden, s.features};
  p.dw_extent[2] = {s.features, s.hidden};
  p.grad = make_plan(&eh, 1, ceil_div(s.features, ffn::kStepK), false,
                     ffn_saved_planes(s) == 1);
  if (ffn_saved_planes(s) == 1) p.grad.bn = 256;  // REGRAD has one width
  p.dx = make_plan(&ex, 1, 2 * ceil_div(s.hidden, ffn::kStepK), true, false);
  p.dw = make_plan(p.dw_extent, 3, ceil_div(s.rows, ffn::kStepK), true, false);
  p.dg = take_rows(c, s.rows, s.hidden);
  p.du = take_rows(c, s.rows, s.hidden);
  if (p.pad_d) {
    p.dy = take_rows(c, s.rows, s.features);
    p.x = take_rows(c, s.rows, s.features);
    p.w_gate = take_rows(c, s.hidden, s.features);
    p.w_up = take_rows(c, s.hidden, s.features);
    p.out_dx = take_rows(c, s.rows, s.features);
  }
  if (p.pad_f) p.w_down = take_rows(c, s.features, s.hidden);
  for (int i = 0; i < 3; ++i) {
    if (i < 2 ? p.pad_d : p.pad_f) p.out_dw[i] = take_rows(c, p.dw_extent[i].m, p.dw_extent[i].n);
  }
  p.partial = c.take(std::max(p.dx.partial_bytes(), p.dw.partial_bytes()));
  return p;
}

}  // namespace

int ffn_saved_planes(const FfnShape& s) {
  const int64_t tiles = ceil_div(s.rows, 256) * ceil_div(s.hidden, 128);
  return s.features <= kRecomputeFeatures && tiles >= device_sm_count() ? 1 : 4;
}

size_t ffn_plane_bytes(const FfnShape& s) {
  return static_cast<size_t>(s.rows) * padded(s.hidden) * 2;
}

size_t ffn_forward_workspace_bytes(const FfnShape& s, bool save) {
  Carver c{nullptr};
  plan_forward(s, save, c);
  return c.used;
}

size_t ffn_backward_workspace_bytes(const FfnShape& s) {
  Carver c{nullptr};
  plan_backward(s, c);
  return c.used;
}

int launch_ffn_forward(const FfnForward& f, void* ws, cudaStream_t stream) {
  const FfnShape& s = f.shape;
  const int64_t m = s.rows, d = s.features, hid = s.hidden, fp = padded(hid);
  char* saved = static_cast<char*>(f.saved);
  const size_t plane = ffn_plane_bytes(s);
  Carver c{static_cast<char*>(ws)};
  const ForwardPlan p = plan_forward(s, saved != nullptr, c);
  const bool keep = ffn_saved_planes(s) > 1;  // g and u, for the backward pass
  if (m <= kFewRows) {
    void* h = saved != nullptr ? saved : p.h;
    void* planes[3] = {};
    for (int i = 0; i < 3 && saved != nullptr && keep; ++i) planes[i] = saved + (i + 1) * plane;
    return s.dtype == CCV_DTYPE_BF16 ? run_rows<__nv_bfloat16>(f, h, planes, stream)
                                     : run_rows<__half>(f, h, planes, stream);
  }
  const Padded x{f.x, f.x_stride, m, d, p.x}, wg{f.w_gate, d, hid, d, p.w_gate},
      wu{f.w_up, d, hid, d, p.w_up}, wd{f.w_down, hid, d, hid, p.w_down};
  RowCopies copies;
  for (const Padded* q : {&x, &wg, &wu, &wd}) q->fill(copies);
  int rc = copy_rows(copies, stream);
  if (rc != CCV_OK) return rc;
  void* h = saved != nullptr ? saved : p.h;
  {
    Product<ffn::GATE, false, false> g(s.dtype, p.gate, d, s.activation);
    g.operand_a(0, x.matrix());
    g.operand_b(0, wg.matrix());
    g.operand_b(1, wu.matrix());
    g.result(0, h, m, hid, fp);
    if (saved != nullptr && keep) {
      for (int i = 1; i <= 3; ++i) g.plane(&g.prm.out[i], saved + i * plane, m, hid, fp);
      g.prm.save = 1;
    }
    g.problem(0, m, hid);
    if ((rc = g.launch(stream)) != CCV_OK) return rc;
  }
  Product<ffn::PLAIN, false, false> y(s.dtype, p.down, hid, 0);
  y.operand_a(0, {h, hid, m, fp});
  y.operand_b(0, wd.matrix());
  y.problem(0, m, d);
  y.partials(p.partial);
  y.result(0, p.y != nullptr ? p.y : f.y, m, d, p.y != nullptr ? padded(d) : d);
  if ((rc = y.launch(stream)) != CCV_OK || p.y == nullptr) return rc;
  RowCopies out;
  out.add(p.y, padded(d), f.y, d, m, d);
  return copy_rows(out, stream);
}

int launch_ffn_backward(const FfnBackward& b, void* ws, cudaStream_t stream) {
  const FfnShape& s = b.shape;
  const int64_t m = s.rows, d = s.features, hid = s.hidden, fp = padded(hid);
  const size_t plane = ffn_plane_bytes(s);
  const char* saved = static_cast<const char*>(b.saved);
  void* const dw[3] = {b.dw_gate, b.dw_up, b.dw_down};
  if (m == 0) {
    for (void* w : dw) {
      if (w == nullptr) continue;
      const int rc = launched(cudaMemsetAsync(w, 0, static_cast<size_t>(d) * hid * 2, stream),
                              "cudaMemsetAsync");
      if (rc != CCV_OK) return rc;
    }
    return CCV_OK;
  }
  Carver c{static_cast<char*>(ws)};
  const BackwardPlan p = plan_backward(s, c);
  const bool need_grad = b.dx != nullptr || dw[0] != nullptr || dw[1] != nullptr;
  const Padded dy{b.dy, b.dy_stride, m, d, p.dy}, x{b.x, b.x_stride, m, d, p.x},
      wg{b.w_gate, d, hid, d, p.w_gate}, wu{b.w_up, d, hid, d, p.w_up},
      wd{b.w_down, hid, d, hid, p.w_down};
  RowCopies copies, out_copies;
  dy.fill(copies);
  const bool recompute = ffn_saved_planes(s) == 1;
  if (recompute || dw[0] != nullptr || dw[1] != nullptr) x.fill(copies);
  if (need_grad) wd.fill(copies);
  if (b.dx != nullptr || (need_grad && recompute)) {
    wg.fill(copies);
    wu.fill(copies);
  }
  int rc = copy_rows(copies, stream);
  if (rc != CCV_OK) return rc;
  if (need_grad && recompute) {
    Product<ffn::REGRAD, false, false> g(s.dtype, p.grad, d, s.activation);
    g.prm.segments = 2;
    g.operand_a(0, dy.matrix());
    g.operand_a(1, x.matrix());
    g.operand_b(0, wg.matrix());
    g.operand_b(1, wu.matrix());
    if (g.rc == CCV_OK) {
      const Matrix w = wd.matrix();
      g.rc = encode_2d(&g.prm.b[2], s.dtype, w.base, w.inner, w.outer, w.ld, 64, 64);
    }
    g.result(0, p.dg, m, hid, fp);
    g.result(1, p.du, m, hid, fp);
    g.problem(0, m, hid);
    if ((rc = g.launch(stream)) != CCV_OK) return rc;
  } else if (need_grad) {
    Product<ffn::GRAD, false, true> g(s.dtype, p.grad, d, s.activation);
    g.operand_a(0, dy.matrix());
    g.operand_b(0, wd.matrix());
    g.result(0, p.dg, m, hid, fp);
    g.result(1, p.du, m, hid, fp);
    for (int i = 0; i < 3; ++i) g.plane(&g.prm.in[i], saved + (i + 1) * plane, m, hid, fp);
    g.problem(0, m, hid);
    if ((rc = g.launch(stream)) != CCV_OK) return rc;
  }
  if (b.dx != nullptr) {
    Product<ffn::PLAIN, false, true> g(s.dtype, p.dx, hid, 0);
    g.prm.segments = 2;
    g.operand_a(0, {p.dg, hid, m, fp});
    g.operand_a(1, {p.du, hid, m, fp});
    g.operand_b(0, wg.matrix());
    g.operand_b(1, wu.matrix());
    g.problem(0, m, d);
    void* out = p.out_dx != nullptr ? p.out_dx : b.dx;
    g.result(0, out, m, d, p.out_dx != nullptr ? padded(d) : d);
    g.partials(p.partial);
    if ((rc = g.launch(stream)) != CCV_OK) return rc;
    if (p.out_dx != nullptr) out_copies.add(out, padded(d), b.dx, d, m, d);
  }
  const Matrix left[3] = {{p.dg, hid, m, fp}, {p.du, hid, m, fp}, dy.matrix()};
  const Matrix right[3] = {x.matrix(), x.matrix(), {saved, hid, m, fp}};
  Product<ffn::PLAIN, true, true> g(s.dtype, p.dw, m, 0);
  int count = 0;
  for (int i = 0; i < 3; ++i) {
    if (dw[i] == nullptr) continue;
    const Extent& e = p.dw_extent[i];
    g.operand_a(count, left[i]);
    g.operand_b(count, right[i]);
    g.problem(count, e.m, e.n);
    void* out = p.out_dw[i] != nullptr ? p.out_dw[i] : dw[i];
    g.result(count, out, e.m, e.n, p.out_dw[i] != nullptr ? padded(e.n) : e.n);
    ++count;
  }
  if (count > 0) {
    g.partials(p.partial);
    if ((rc = g.launch(stream)) != CCV_OK) return rc;
  }
  for (int i = 0; i < 3; ++i) {
    if (dw[i] == nullptr || p.out_dw[i] == nullptr) continue;
    const Extent& e = p.dw_extent[i];
    out_copies.add(p.out_dw[i], padded(e.n), dw[i], e.n, e.m, e.n);
  }
  return copy_rows(out_copies, stream);
}

}  // namespace ccv
