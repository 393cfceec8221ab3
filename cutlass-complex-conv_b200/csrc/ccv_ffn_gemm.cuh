// Matrix products of the gated feed-forward block on tcgen05, one persistent
// kernel template for all of them:
//   GATE   h = act(x Wg^T) (x Wu^T)        epilogue: activation and product
//   PLAIN  c = a b (+ a' b')               down projection, dx, weight gradients
//   GRAD   dh = dy Wd                      epilogue: dg, du from dh and the g, u kept
//   REGRAD g, u as GATE, dh as GRAD        epilogue: dg, du; nothing was kept of g, u
//
// A cluster of two CTAs computes a tile of 256 x BN with
// tcgen05.mma.cta_group::2: each CTA holds 128 rows of A and half of B's BN
// columns in shared memory and its 128 rows of the fp32 sums in TMEM.  Per
// K step of 64 a CTA loads 16 KB of A and 64 BN bytes of B (TMA, 128-byte
// swizzle).  For GATE, one CTA's half of B is the gate projection's rows and
// the other's the up projection's, so the sums of g and u of one output lie
// in the same TMEM lane, BN / 2 columns apart, and the epilogue needs no
// exchange.  Operands whose reduction index is not innermost in memory (the
// weights in dh and dx, both operands of the weight gradients) are loaded as
// they lie and multiplied through the M/N-innermost descriptor form: nothing
// is transposed.
//
// Measured on B200 at 8192 x 2048 x 8192 bf16, isolated launches: GATE 331 us
// (1.66 PFLOP/s; cuBLAS bf16 burst 1.69), down 172, dx 336, the three weight
// gradients 508 (1.62), GRAD 245 (1.12: its planes' traffic and epilogue);
// back to back the power cap lowers the clock to about 1.3 PFLOP/s.
//
// Two accumulators in TMEM let the epilogue warps work on one tile while
// the next is multiplied; they pass their results through swizzled
// shared-memory slots to TMA stores, which clip the ragged edges.
//
// Warps: 0 TMA producer, 1 TMEM allocation and MMA issue (even CTA), then the
// epilogue (quarter of the rows = warp % 4, a group of the columns).
#pragma once

#include <cuda.h>

#include "ccv_internal.h"
#include "ccv_ptx.cuh"
#include "ccv_tokens.cuh"

namespace ccv {
namespace ffn {

enum Mode { GATE, PLAIN, GRAD, REGRAD };

constexpr int kRows = 128;        // rows of one CTA's tile
constexpr int kStepK = 64;        // reduction elements per pipeline stage: 128-byte rows
constexpr int kOperandA = kRows * kStepK * 2;
constexpr int kMaxProblems = 3;
constexpr int kRasterRows = 8;    // tile rows walked together (operand reuse in L2)
constexpr int kTimeoutCode = CCV_ERR_DEVICE_TIMEOUT;

struct Tiles {
  int m, n;              // extents of the result
  int tiles_m, tiles_n;
  int first;             // first tile
  uint32_t band_inverse; // floor(2^32 / (kRasterRows * tiles_n))
};

struct alignas(64) GemmParams {
  // One problem: segments of the reduction, a[s] with b[s] (GATE: b[0] gate
  // rows, b[1] up rows).  Several problems: one segment each.
  CUtensorMap a[kMaxProblems], b[kMaxProblems];
  CUtensorMap out[4];  // GATE: h and (saving) the three planes of g and u; GRAD: dg, du;
                       // PLAIN: per problem
  CUtensorMap in[3];   // GRAD: the planes of g and u
  CUtensorMap partial;            // split tiles: fp32 [tile part][256][BN]
  Tiles tiles[kMaxProblems];
  int* status;
  int problems, segments;
  int ksteps;   // per segment
  // Work units: tiles 0 .. whole - 1, then the other tiles in `splits` parts
  // of the reduction each (PLAIN), whose partial sums ffn_split_sum adds.
  int whole, splits;
  int units;
  int save;     // GATE: store g and u too
};

template <int MODE, int BN>
struct Config {
  static constexpr int kOperandB = BN / 2 * kStepK * 2;
  static constexpr int kStage = kOperandA + kOperandB;
  // The gate epilogue is bound by issue slots and latency: sixteen warps work
  // on a 256-wide tile (39 -> 35 us at 25088 x 256 -> 2 x 1024 GELU).
  static constexpr int kEpiWarps = (MODE == GATE || MODE == REGRAD) && BN == 256 ? 16 : 8;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kGroups = kEpiWarps / 4;  // warps that share a row quarter's columns
  // BN = 256: one block per SM.  BN = 128, for problems of few tiles: few
  // stages and little staging, so that two blocks share an SM and the next
  // launch's blocks start up beside this one's.  GRAD trades a stage for room
  // to load its inputs a chunk ahead.
  static constexpr int kBlocksPerSm = BN == 256 || MODE == GRAD ? 1 : 2;
  static constexpr int kStaging = MODE == GRAD ? 98304 : (BN == 256 ? 65536 : 32768);
  static constexpr int kWarpStaging = kStaging / kEpiWarps;
  static constexpr int kStages = MODE == GRAD ? (BN == 256 ? 4 : 5) : (BN == 256 ? 5 : 3);
  static constexpr int kStagingOffset = kStages * kStage;
  static constexpr int kBarOffset = kStagingOffset + kStaging;
  static constexpr int kBarBytes = 512;
  static constexpr int kSmem = kBarOffset + kBarBytes + 1024;
  // REGRAD: one accumulator of BN columns for g and u, two of BN / 2 for dh.
  static constexpr int kAccumulators = MODE == REGRAD ? 1 : 2;
  static constexpr int kTmemCols = 2 * BN;
  static_assert(kSmem <= 232448, "shared memory");
  static_assert((2 * kStages + 5 + 2 * kEpiWarps) * 8 + 16 <= kBarBytes, "barriers");
};

struct Unit {
  int problem, tm, tn, k0, k1;
  int part;  // index among the split tiles' parts, -1: a whole tile
};

// Problem, tile row and tile column of a tile.
__device__ __forceinline__ void locate(const Tiles* tiles, int problems, int tile, int& problem,
                                       int& tm, int& tn) {
  problem = 0;
  for (int i = 1; i < kMaxProblems; ++i) {
    if (i < problems && tile >= tiles[i].first) problem = i;
  }
  const Tiles& t = tiles[problem];
  // Bands of kRasterRows tile rows, walked column by column.  The quotient by
  // the inverse is exact or one too small.
  const uint32_t local = static_cast<uint32_t>(tile - t.first);
  const uint32_t size = static_cast<uint32_t>(kRasterRows * t.tiles_n);
  uint32_t band = __umulhi(local, t.band_inverse);
  uint32_t r = local - band * size;
  if (r >= size) {
    ++band;
    r -= size;
  }
  const int left = t.tiles_m - static_cast<int>(band) * kRasterRows;
  if (left >= kRasterRows) {
    tn = static_cast<int>(r / kRasterRows);
    tm = static_cast<int>(band * kRasterRows + r % kRasterRows);
  } else {
    tn = static_cast<int>(r) / left;
    tm = static_cast<int>(band) * kRasterRows + static_cast<int>(r) - tn * left;
  }
}

__device__ __forceinline__ Unit decode(const GemmParams& p, int u) {
  Unit w;
  const int total = p.ksteps * p.segments;
  int tile = u;
  w.part = -1;
  w.k0 = 0;
  w.k1 = total;
  if (u >= p.whole) {
    w.part = u - p.whole;
    const int q = w.part / p.splits;
    const int s = w.part - q * p.splits;
    tile = p.whole + q;
    w.k0 = static_cast<int>(static_cast<long long>(total) * s / p.splits);
    w.k1 = static_cast<int>(static_cast<long long>(total) * (s + 1) / p.splits);
  }
  locate(p.tiles, p.problems, tile, w.problem, w.tm, w.tn);
  return w;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// act(g) and act'(g).  The sigmoid is two hardware approximations (2^x and
// 1/x, a few 2^-23 each): a relative error far below the 16-bit rounding of
// the result.  GELU's normal distribution is Abramowitz and Stegun 7.1.26, a
// polynomial times exp(-g^2/2), the exponential its slope needs too.  Its
// bound is an absolute one (|error of erf| <= 1.5e-7, and a few 2^-24), so in
// the lower tail the relative error passes the result's rounding: 1.9e-4 at
// g = -3.5, 4.7e-4 at -4 (half a step of float16 is 4.9e-4, of bfloat16
// 3.9e-3), 1.6e-3 at -5, 3.6e-3 at -6, of values from 8e-4 down.  (A float32
// 1 + erf(g / sqrt 2) loses more to cancellation from -5 on.)
template <int ACT>
__device__ __forceinline__ void activation(float g, float& value, float& slope) {
  if constexpr (ACT == CCV_ACTIVATION_SILU) {
    const float s = rcp(1.f + ex2(g * -1.4426950408889634f));
    value = g * s;
    slope = fmaf(-value, s, value) + s;
  } else {
    const float t = rcp(fmaf(0.3275911f * 0.70710678118654752f, fabsf(g), 1.f));
    const float e = ex2(g * g * (-0.5f * 1.4426950408889634f));
    float q = fmaf(t, 1.061405429f, -1.453152027f);
    q = fmaf(t, q, 1.421413741f);
    q = fmaf(t, q, -0.284496736f);
    q = fmaf(t, q, 0.254829592f);
    const float tail = 0.5f * t * q * e;
    const float c = g >= 0.f ? 1.f - tail : tail;
    value = g * c;
    slope = fmaf(g * 0.39894228040143268f, e, c);
  }
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// g and u kept for the backward pass, to 24 bits of float32 each (a relative step
// of 2^-15; 16 bits of either would show in dx and in the weight gradients
// beside the roundings of dg and of the result): planes of the high 16 bits
// of g, of u, and of the next 8 bits of both (g's in the low byte).
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {
  return __byte_perm(a, b, 0x7632);
}
__device__ __forceinline__ uint32_t next_bytes(uint32_t g0, uint32_t u0, uint32_t g1, uint32_t u1) {
  return __byte_perm(__byte_perm(g0, u0, 0x0051), __byte_perm(g1, u1, 0x0051), 0x5410);
}
// The values of one plane word (two elements) and their word of next bytes;
// the lowest byte repeats the next one, below the 24 bits.
__device__ __forceinline__ float2 unpack_g(uint32_t high, uint32_t next) {
  return make_float2(__uint_as_float(__byte_perm(high, next, 0x1044)),
                     __uint_as_float(__byte_perm(high, next, 0x3266)));
}
__device__ __forceinline__ float2 unpack_u(uint32_t high, uint32_t next) {
  return make_float2(__uint_as_float(__byte_perm(high, next, 0x1055)),
                     __uint_as_float(__byte_perm(high, next, 0x3277)));
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                             uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// 16-byte unit `j` of row `row` of a slot with 64- or 128-byte rows, where
// TMA's swizzle of that width puts it.
__device__ __forceinline__ uint32_t slot64(uint32_t slot, int row, int j) {
  return slot + row * 64 + ((j ^ ((row >> 1) & 3)) << 4);
}
__device__ __forceinline__ uint32_t slot128(uint32_t slot, int row, int j) {
  return slot + row * 128 + ((j ^ (row & 7)) << 4);
}

// An epilogue warp's ring of staging slots of BYTES each, written by its
// lanes and read by TMA stores.
template <int TOTAL, int BYTES>
struct Ring {
  static constexpr int kSlots = TOTAL / BYTES;
  uint32_t base;
  uint32_t next = 0;
  // A slot no store still reads.
  __device__ __forceinline__ uint32_t take(int lane) {
    if (lane == 0) ptx::bulk_wait_read_le<kSlots - 1>();
    __syncwarp();
    const uint32_t s = base + (next % kSlots) * BYTES;
    ++next;
    return s;
  }
};

// Makes the lanes' slot writes visible to the async proxy; then lane 0 stores.
__device__ __forceinline__ void publish() {
  ptx::fence_proxy_async_shared();
  __syncwarp();
}

// ACT is a template parameter because a branch on it at each element kept the
// compiler from interleaving elements: the gate epilogue took twice as long.
template <typename T, int MODE, int BN, bool A_MN, bool B_MN, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Config<MODE, BN>::kThreads, Config<MODE, BN>::kBlocksPerSm)
    ffn_gemm_kernel(const __grid_constant__ GemmParams p) {
  using C = Config<MODE, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
  // full[S] (even CTA), empty[S], tfull[2], tempty[2] (even CTA), done,
  // loaded[2][8] (GRAD: an epilogue warp's g and u), the TMEM address, flags.
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * C::kStages + 5 + 2 * C::kEpiWarps);
  volatile int* flags = reinterpret_cast<volatile int*>(tmem_holder + 1);  // [0] skip, [1] abort

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const bool leader = rank == 0;
  const int cid = static_cast<int>(ptx::cluster_id_x());
  const int ncl = static_cast<int>(ptx::nclusters_x());
  const uint32_t smem_base = ptx::smem_u32(smem);
  const uint32_t bar_base = ptx::smem_u32(bars);
  auto full_bar = [&](int i) { return bar_base + 8u * i; };
  auto empty_bar = [&](int i) { return bar_base + 8u * (C::kStages + i); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * C::kStages + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * C::kStages + 2 + b); };
  const uint32_t done_bar = bar_base + 8u * (2 * C::kStages + 4);
  const uint32_t loaded_bar0 = bar_base + 8u * (2 * C::kStages + 5);

  if (threadIdx.x == 0) {
    flags[1] = 0;
    for (int i = 0; i < C::kStages; ++i) {
      ptx::mbar_init(full_bar(i), 1);
      ptx::mbar_init(empty_bar(i), 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(tfull_bar(b), 1);
      ptx::mbar_init(tempty_bar(b), 2 * C::kEpiWarps);  // both CTAs' epilogue warps
    }
    ptx::mbar_init(done_bar, 1);
    for (int i = 0; i < 2 * C::kEpiWarps; ++i) ptx::mbar_init(loaded_bar0 + 8u * i, 1);
    ptx::fence_mbar_init();
  }
  // A timeout reported by an earlier kernel: this one exits without work.
  if (threadIdx.x == 32) flags[0] = *reinterpret_cast<volatile int*>(p.status) != 0 ? 1 : 0;
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&p.a[0]);
    ptx::prefetch_tmap(&p.b[MODE == GATE || MODE == REGRAD ? rank : 0]);
    ptx::prefetch_tmap(&p.out[0]);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(ptx::smem_u32(tmem_holder), C::kTmemCols);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  // Everything above may overlap the previous kernel on the stream.
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const uint32_t tmem_base = *tmem_holder;
  const bool skip = flags[0] != 0;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    // The whole warp walks the loop, so that addresses and coordinates stay
    // in uniform registers, and one lane issues: with a loop of one lane alone
    // a K step took 0.47 us to issue, more than its multiplication.
    if (!skip) {
      const bool issuer = ptx::elect_one() != 0;
      const uint32_t lead_full = ptx::mapa_shared(full_bar(0), 0);
      uint32_t stage = 0, parity = 1, issued = 0;
      bool abort = false;
      for (int u = cid; u < p.units && !abort; u += ncl) {
        const Unit w = decode(p, u);
        const int m0 = (2 * w.tm + static_cast<int>(rank)) * kRows;
        constexpr bool kGated = MODE == GATE || MODE == REGRAD;  // BN / 2 outputs a tile
        const int n0 = kGated ? w.tn * (BN / 2) : w.tn * BN + static_cast<int>(rank) * (BN / 2);
        for (int seg = 0; seg < p.segments && !abort; ++seg) {
          const int first = max(w.k0 - seg * p.ksteps, 0);
          const int last = min(w.k1 - seg * p.ksteps, p.ksteps);
          const int map = p.problems > 1 ? w.problem : seg;
          const CUtensorMap* ma = &p.a[map];
          // REGRAD's first segment is dh: dy with the down projection, whose
          // hidden index is innermost, half of the tile's outputs per CTA.
          const bool down = MODE == REGRAD && seg == 0;
          const CUtensorMap* mb = &p.b[down ? 2 : (kGated ? static_cast<int>(rank) : map)];
          for (int ks = first; ks < last; ++ks) {
            if (!ptx::mbar_wait_bounded(empty_bar(stage), parity, p.status, kTimeoutCode)) {
              flags[1] = 1;
              abort = true;
              break;
            }
            const uint32_t fb = lead_full + 8u * stage;
            const uint32_t sa = smem_base + stage * C::kStage;
            const uint32_t sb = sa + kOperandA;
            const int k = ks * kStepK;
            if (issuer) {
              if (leader) {
                ptx::mbar_arrive_expect_tx(full_bar(stage),
                                           2 * (down ? kOperandA + 8192 : C::kStage));
              }
              if constexpr (A_MN) {
                ptx::tma_load_2d_pair(sa, ma, fb, m0, k);
                ptx::tma_load_2d_pair(sa + 8192, ma, fb, m0 + 64, k);
              } else {
                ptx::tma_load_2d_pair(sa, ma, fb, k, m0);
              }
              if constexpr (B_MN) {
#pragma unroll
                for (int i = 0; i < BN / 128; ++i) {
                  ptx::tma_load_2d_pair(sb + 8192 * i, mb, fb, n0 + 64 * i, k);
                }
              } else if (down) {
                ptx::tma_load_2d_pair(sb, mb, fb, n0 + static_cast<int>(rank) * 64, k);
              } else {
                ptx::tma_load_2d_pair(sb, mb, fb, k, n0);
              }
            }
            ++issued;
            if (++stage == C::kStages) {
              stage = 0;
              parity ^= 1u;
            }
          }
        }
      }
      if (leader) {
        // Drain: every issued stage's bytes (both CTAs) have landed.
        for (uint32_t j = 0; j < static_cast<uint32_t>(C::kStages) && j < issued; ++j) {
          const uint32_t gg = issued - 1 - j;
          ptx::mbar_wait_bounded(full_bar(static_cast<int>(gg % C::kStages)),
                                 (gg / C::kStages) & 1u, p.status, kTimeoutCode);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    if (leader && !skip) {
      constexpr uint32_t idesc = ptx::idesc_f16(2 * kRows, BN, kIsBf16<T>, A_MN, B_MN);
      const bool issuer = ptx::elect_one() != 0;
      // Descriptors of stage 0; a stage or K step further is an addition to
      // the address field (16-byte units).
      const uint64_t da0 = A_MN ? ptx::desc_mnmajor_sw128(smem_base, 8192)
                                : ptx::desc_kmajor_sw128(smem_base);
      const uint64_t db0 = B_MN ? ptx::desc_mnmajor_sw128(smem_base + kOperandA, 8192)
                                : ptx::desc_kmajor_sw128(smem_base + kOperandA);
      constexpr uint32_t kStepA = (A_MN ? 2048 : 32) / 16, kStepB = (B_MN ? 2048 : 32) / 16;
      uint32_t stage = 0, parity = 0;
      int i = 0;
      bool abort = false;
      for (int u = cid; u < p.units && !abort; u += ncl, ++i) {
        const Unit w = decode(p, u);
        const int buf = i % C::kAccumulators;
        auto wait_free = [&]() {
          const bool free = ptx::mbar_wait_bounded(
              tempty_bar(buf), ((i / C::kAccumulators) & 1u) ^ 1u, p.status, kTimeoutCode);
          if (!free) flags[1] = 1;
          ptx::tc_fence_after();
          return free;
        };
        // REGRAD multiplies dh into the buffer of the tile before last (whose
        // epilogue was waited for then) while the last tile's is at work, and
        // waits before g and u.
        if (MODE != REGRAD && !wait_free()) break;
        const uint32_t d = tmem_base + static_cast<uint32_t>(buf * BN);
        for (int ks = w.k0; ks < w.k1; ++ks) {
          if (!ptx::mbar_wait_bounded(full_bar(stage), parity, p.status, kTimeoutCode)) {
            flags[1] = 1;
            abort = true;
            break;
          }
          ptx::tc_fence_after();
          if (MODE == REGRAD && ks == p.ksteps && !wait_free()) {
            abort = true;
            break;
          }
          const uint64_t da = da0 + stage * (C::kStage / 16);
          const uint64_t db = db0 + stage * (C::kStage / 16);
          if (MODE == REGRAD && ks < p.ksteps) {
            if (issuer) {
              constexpr uint32_t down = ptx::idesc_f16(2 * kRows, BN / 2, kIsBf16<T>, false, true);
              const uint64_t dw =
                  ptx::desc_mnmajor_sw128(smem_base + kOperandA, 8192) + stage * (C::kStage / 16);
#pragma unroll
              for (int kk = 0; kk < kStepK / 16; ++kk) {
                ptx::mma_f16_pair(d + BN + (i & 1) * (BN / 2), da + kk * kStepA,
                                  dw + kk * (2048 / 16), down, (ks != 0 || kk != 0) ? 1u : 0u);
              }
              ptx::mma_commit_pair(empty_bar(stage));
            }
          } else if (issuer) {
#pragma unroll
            for (int kk = 0; kk < kStepK / 16; ++kk) {
              ptx::mma_f16_pair(d, da + kk * kStepA, db + kk * kStepB, idesc,
                                (ks != (MODE == REGRAD ? p.ksteps : w.k0) || kk != 0) ? 1u : 0u);
            }
            ptx::mma_commit_pair(empty_bar(stage));
          }
          if (++stage == C::kStages) {
            stage = 0;
            parity ^= 1u;
          }
        }
        if (issuer) ptx::mma_commit_pair(tfull_bar(buf));
      }
      // All issued MMAs complete before teardown.
      if (issuer) ptx::mma_commit_pair(done_bar);
      ptx::mbar_wait_bounded(done_bar, 0, p.status, kTimeoutCode);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int e = warp - 2;
    const int quarter = warp & 3;
    const int group = e >> 2;  // of the columns
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t staging = smem_base + C::kStagingOffset + e * C::kWarpStaging;
    const uint32_t loaded = loaded_bar0 + 16u * e;
    const uint32_t tempty0 = ptx::mapa_shared(tempty_bar(0), 0);
    const uint32_t tempty1 = ptx::mapa_shared(tempty_bar(1), 0);
    Ring<C::kWarpStaging, 2048> ring2{staging};
    Ring<C::kWarpStaging, 4096> ring4{staging};
    uint32_t loads = 0, loads_issued = 0;
    int i = 0;
    for (int u = cid; u < p.units && !skip; u += ncl, ++i) {
      const Unit w = decode(p, u);
      const Tiles& t = p.tiles[w.problem];
      const int buf = i % C::kAccumulators;
      const uint32_t use = static_cast<uint32_t>(i / C::kAccumulators);
      const int row0 = (2 * w.tm + static_cast<int>(rank)) * kRows + quarter * 32;
      const bool rows_in = row0 < t.m;
      const uint32_t acc = t_row + static_cast<uint32_t>(buf * BN);
      // GRAD: the planes of g and u, 32 columns at a time, loaded a chunk ahead
      // into two alternating slots (the first during the mainloop); dg and du
      // replace the high halves there and are stored from there.
      constexpr int kGradChunks = BN / 2 / 32;
      constexpr uint32_t kGradBytes = 3 * 2048, kGradSlots = 2;
      const int grad_col = w.tn * BN + group * (BN / 2);
      auto load_inputs = [&](int c) {
        if (lane == 0) {
          ptx::bulk_wait_read_all();  // the slot's last results have been read
          const uint32_t slot = staging + (loads_issued % kGradSlots) * kGradBytes;
          const uint32_t bar = loaded + 8u * (loads_issued % kGradSlots);
          ptx::mbar_arrive_expect_tx(bar, kGradBytes);
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            ptx::tma_load_2d(slot + 2048 * i, &p.in[i], bar, grad_col + 32 * c, row0);
          }
        }
        ++loads_issued;
      };
      if constexpr (MODE == GRAD) load_inputs(0);
      bool ok = ptx::mbar_wait_bounded_backoff(tfull_bar(buf), use & 1u, p.status, kTimeoutCode);
      ptx::tc_fence_after();
      if (!ok) flags[1] = 1;
      const bool store = ok && !flags[1];
      // This warp has read its part of the accumulator: the MMA issuer may
      // overwrite it once every epilogue warp says so.
      auto release = [&]() {
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster_relaxed(buf == 0 ? tempty0 : tempty1);
      };
      if constexpr (MODE == GATE) {
        static_assert(BN / 2 / C::kGroups == 32, "32 outputs per warp");
        const int fc = group * 32;
        uint32_t g[32], v[32];
        ptx::tmem_ld_32x32b_x32(acc + fc, g);
        ptx::tmem_ld_32x32b_x32(acc + BN / 2 + fc, v);
        ptx::tmem_wait_ld();
        ptx::reg_fence(g);
        ptx::reg_fence(v);
        release();
        const int col = w.tn * (BN / 2) + fc;
        const bool in = store && rows_in && col < t.n;
        // word(k): elements 2 k and 2 k + 1.
        auto put = [&](auto&& word, const CUtensorMap* map) {
          const uint32_t slot = ring2.take(lane);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            st_shared_v4(slot64(slot, lane, j), word(4 * j), word(4 * j + 1), word(4 * j + 2),
                         word(4 * j + 3));
          }
          publish();
          if (lane == 0) {
            if (in) ptx::tma_store_2d(map, slot, col, row0);
            ptx::bulk_commit_group();
          }
        };
        put([&](int k) {
          float v0, v1, slope;
          activation<ACT>(__uint_as_float(g[2 * k]), v0, slope);
          activation<ACT>(__uint_as_float(g[2 * k + 1]), v1, slope);
          return pack2(v0 * __uint_as_float(v[2 * k]), v1 * __uint_as_float(v[2 * k + 1]), T());
        }, &p.out[0]);
        if (p.save) {
          put([&](int k) { return high_halves(g[2 * k], g[2 * k + 1]); }, &p.out[1]);
          put([&](int k) { return high_halves(v[2 * k], v[2 * k + 1]); }, &p.out[2]);
          put([&](int k) { return next_bytes(g[2 * k], v[2 * k], g[2 * k + 1], v[2 * k + 1]); },
              &p.out[3]);
        }
      } else if constexpr (MODE == REGRAD) {
        // 32 outputs per warp, 16 at a time (three values each).
        const int fc = group * 32;
        const int col = w.tn * (BN / 2) + fc;
        const uint32_t dg_slot = ring2.take(lane), du_slot = ring2.take(lane);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t g[16], v[16], d[16];
          ptx::tmem_ld_32x32b_x16(acc + fc + h * 16, g);
          ptx::tmem_ld_32x32b_x16(acc + BN / 2 + fc + h * 16, v);
          ptx::tmem_ld_32x32b_x16(acc + BN + (i & 1) * (BN / 2) + fc + h * 16, d);
          ptx::tmem_wait_ld();
          ptx::reg_fence(g);
          ptx::reg_fence(v);
          ptx::reg_fence(d);
          if (h == 1) release();
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t og[4], ou[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int at = 8 * j + 2 * k;
              float v0, s0, v1, s1;
              activation<ACT>(__uint_as_float(g[at]), v0, s0);
              activation<ACT>(__uint_as_float(g[at + 1]), v1, s1);
              const float d0 = __uint_as_float(d[at]), d1 = __uint_as_float(d[at + 1]);
              og[k] = pack2(d0 * __uint_as_float(v[at]) * s0, d1 * __uint_as_float(v[at + 1]) * s1,
                            T());
              ou[k] = pack2(d0 * v0, d1 * v1, T());
            }
            st_shared_v4(slot64(dg_slot, lane, 2 * h + j), og[0], og[1], og[2], og[3]);
            st_shared_v4(slot64(du_slot, lane, 2 * h + j), ou[0], ou[1], ou[2], ou[3]);
          }
        }
        publish();
        if (lane == 0) {
          if (store && rows_in && col < t.n) {
            ptx::tma_store_2d(&p.out[0], dg_slot, col, row0);
            ptx::tma_store_2d(&p.out[1], du_slot, col, row0);
          }
          ptx::bulk_commit_group();
          ptx::bulk_commit_group();  // one group per slot of the ring
        }
      } else if constexpr (MODE == GRAD) {
#pragma unroll 1
        for (int c = 0; c < kGradChunks; ++c) {
          if (c + 1 < kGradChunks) load_inputs(c + 1);
          const int col = grad_col + c * 32;
          const uint32_t slot = staging + (loads % kGradSlots) * kGradBytes;
          uint32_t d[32];
          ptx::tmem_ld_32x32b_x32(acc + group * (BN / 2) + c * 32, d);
          ok = ptx::mbar_wait_bounded(loaded + 8u * (loads % kGradSlots), (loads / kGradSlots) & 1u,
                                              p.status, kTimeoutCode) && ok;
          ++loads;
          if (!ok) flags[1] = 1;
          ptx::tmem_wait_ld();
          ptx::reg_fence(d);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t ag = slot64(slot, lane, j);
            const uint32_t au = slot64(slot + 2048, lane, j);
            const uint4 g4 = ld_shared_v4(ag), u4 = ld_shared_v4(au);
            const uint4 n4 = ld_shared_v4(slot64(slot + 4096, lane, j));
            const uint32_t gw[4] = {g4.x, g4.y, g4.z, g4.w}, uw[4] = {u4.x, u4.y, u4.z, u4.w};
            const uint32_t nw[4] = {n4.x, n4.y, n4.z, n4.w};
            uint32_t og[4], ou[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 gg = unpack_g(gw[k], nw[k]), uu = unpack_u(uw[k], nw[k]);
              const float d0 = __uint_as_float(d[8 * j + 2 * k]);
              const float d1 = __uint_as_float(d[8 * j + 2 * k + 1]);
              float v0, s0, v1, s1;
              activation<ACT>(gg.x, v0, s0);
              activation<ACT>(gg.y, v1, s1);
              og[k] = pack2(d0 * uu.x * s0, d1 * uu.y * s1, T());
              ou[k] = pack2(d0 * v0, d1 * v1, T());
            }
            st_shared_v4(ag, og[0], og[1], og[2], og[3]);
            st_shared_v4(au, ou[0], ou[1], ou[2], ou[3]);
          }
          publish();
          if (lane == 0) {
            if (ok && !flags[1] && rows_in && col < t.n) {
              ptx::tma_store_2d(&p.out[0], slot, col, row0);
              ptx::tma_store_2d(&p.out[1], slot + 2048, col, row0);
            }
            ptx::bulk_commit_group();
          }
        }
      } else if (w.part >= 0) {
        // fp32 partial sums, 32 columns at a time.
#pragma unroll 1
        for (int c = 0; c < BN / 2; c += 32) {
          uint32_t d[32];
          ptx::tmem_ld_32x32b_x32(acc + group * (BN / 2) + c, d);
          ptx::tmem_wait_ld();
          ptx::reg_fence(d);
          const uint32_t slot = ring4.take(lane);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            st_shared_v4(slot128(slot, lane, j), d[4 * j], d[4 * j + 1], d[4 * j + 2], d[4 * j + 3]);
          }
          publish();
          if (lane == 0) {
            if (store && rows_in) {
              ptx::tma_store_3d(&p.partial, slot, group * (BN / 2) + c,
                                static_cast<int>(rank) * kRows + quarter * 32, w.part);
            }
            ptx::bulk_commit_group();
          }
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < BN / 2; c += 64) {
          const int col = w.tn * BN + group * (BN / 2) + c;
          const uint32_t slot = ring4.take(lane);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t d[32];
            ptx::tmem_ld_32x32b_x32(acc + group * (BN / 2) + c + h * 32, d);
            ptx::tmem_wait_ld();
            ptx::reg_fence(d);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t q[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                q[k] = pack2(__uint_as_float(d[8 * j + 2 * k]),
                             __uint_as_float(d[8 * j + 2 * k + 1]), T());
              }
              st_shared_v4(slot128(slot, lane, h * 4 + j), q[0], q[1], q[2], q[3]);
            }
          }
          publish();
          if (lane == 0) {
            if (store && rows_in && col < t.n) ptx::tma_store_2d(&p.out[w.problem], slot, col, row0);
            ptx::bulk_commit_group();
          }
        }
      }
      if constexpr (MODE == PLAIN || MODE == GRAD) release();
      if (!ok) break;
    }
    // Output stores still in flight complete before the CTA exits.
    if (lane == 0) ptx::bulk_wait_all();
  }

  ptx::cta_sync();
  if (flags[1]) ptx::nanosleep(100000);  // let stray copies of an aborted tile land
  ptx::tc_fence_before();
  ptx::cluster_sync();
  if (warp == 1) {
    __syncwarp();  // tcgen05.dealloc is warp-collective
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem_base, C::kTmemCols);
  }
}

}  // namespace ffn
}  // namespace ccv
