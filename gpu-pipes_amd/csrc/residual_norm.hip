// The norms around a block with its residual: one pass over the rows of
//   h   = x + scale * act(gate) * Post(y)
//   out = Pre(h)
// where Post (of the block that ends) and Pre (of the block that begins) are
// LayerNorm, RMSNorm or nothing.  No counterpart in the reference, whose
// layer norm (common/layer_norm_v2.cuh:129-147) and add
// (common/elemwise_add.cuh:42-54) are kernels of their own.
//
// The bound is memory: x and y are read and h and out written once, 8 bytes a
// value, for some twenty operations.  A row therefore stays in registers from
// its load to its store, and every statistic is taken from there.  16,384 rows
// of 4,096 in bf16: 101 us, 5.3 TB/s (a large copy here: 4.9); 128 of 8,192: 6.0
// us; one of 4,096: 3.5 us, the latencies of a launch, a load and two barriers.
// Rows of an odd length are not aligned to their 16-byte pieces, and cost half
// as much again (16,288 rows of 1,021: 47.5 us, of 1,024: 30 to 34).
#include <hip/hip_runtime.h>

#include "../../include/gpipes.h"
#include "gp_kernels.hpp"
#include "row_ops.hpp"

namespace gp {
namespace {

// Waves whose 64 x 8 values make up one piece of a row; a row is W waves
// wide, each holding C pieces: piece j of wave w is values
// [512 (j W + w), + 512) of the row.
constexpr int kPiece = kWave * 8;
constexpr int kMaxWaves = 16;

// One wave's share of a row's statistics: how many values, their mean, and the
// sum of their squared distances from that mean.
struct Part {
  float n, mean, m2;
};

// LDS for the exchange: [row parity][Post, Pre][wave of the workgroup].
typedef Part Parts[2][2][kMaxWaves];

// Mean and 1 / sqrt(variance + eps) of a row, of which this wave holds the
// values v (kind GP_NORM_RMS: about zero instead of the mean).  Two passes over
// registers give the wave's own mean and squared distances; the waves' parts
// are joined through LDS by the rule for joining two sets,
// M2 = sum(m2) + sum(n (mean_w - mean)^2), one barrier for a norm.  Sums and
// statistics are in 32 bits throughout.  TAIL: a piece of eight may be cut short.
template <int C, bool TAIL>
__device__ __forceinline__ void row_stats(const float (&v)[C][8], const int (&nv)[C], int kind, int D, int W, int w,
                                          float eps, Part* parts, float& mean, float& rstd) {
  Part p{0.f, 0.f, 0.f};
  if (kind == GP_NORM_LAYER) {
    int n = 0;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int left = D - (j * W + w) * kPiece;
      n += left < 0 ? 0 : left > kPiece ? kPiece : left;
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[j][e];  // values past the row's end are zeros
    }
    p.n = (float)n;
    p.mean = n > 0 ? sum_lanes<64>(s) / p.n : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < C; ++j) {
    if (nv[j] <= 0) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = !TAIL || e < nv[j] ? v[j][e] - p.mean : 0.f;
      q = __builtin_fmaf(d, d, q);
    }
  }
  p.m2 = sum_lanes<64>(q);
  if (W > 1) {
    const int lane = threadIdx.x & 63, wb = threadIdx.x >> 6;
    if (lane == 0) parts[wb] = p;
    lds_barrier();
    const int i = lane & 15;
    p = Part{0.f, 0.f, 0.f};
    if (i < W) p = parts[wb - w + i];
    if (kind == GP_NORM_LAYER) {
      const float m = sum_lanes<16>(p.n * p.mean) / (float)D;
      p.m2 = __builtin_fmaf(p.n * (p.mean - m), p.mean - m, p.m2);
      p.mean = m;
    }
    p.m2 = sum_lanes<16>(p.m2);
  }
  mean = p.mean;
  // a precise division and root: once a row, and rsq's last bit would scale every value
  rstd = 1.f / __builtin_sqrtf(p.m2 / (float)D + eps);
}

struct Args {
  ResidualNormArgs a;
  int W;          // waves a row
  int64_t rows;   // consecutive rows a team of W waves takes
  int64_t per;    // rows that share a gate row
};

// A vector over the channels as this thread's lanes need it, in its 16 bits.
template <int C, bool BACK>
__device__ __forceinline__ void load_channels(u32x4 (&u)[C], const half_t* p, const int (&at)[C], const int (&nv)[C],
                                              unsigned none) {
#pragma unroll
  for (int j = 0; j < C; ++j) u[j] = p ? load_raw8<BACK>(p + at[j], nv[j]) : u32x4{none, none, none, none};
}

// (v - mean) rstd gamma + beta over this thread's values (those past the row's end: anything).
template <class T, int C>
__device__ __forceinline__ void affine(float (&v)[C][8], float mean, float rstd, const u32x4 (&gamma)[C],
                                       const u32x4 (&beta)[C], bool add) {
#pragma unroll
  for (int j = 0; j < C; ++j) {
    float g[8];
    widen8<T>(gamma[j], g);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[j][e] = (v[j][e] - mean) * rstd * g[e];
  }
  if (!add) return;
#pragma unroll
  for (int j = 0; j < C; ++j) {
    float b[8];
    widen8<T>(beta[j], b);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[j][e] += b[e];
  }
}

// TAIL: D is no multiple of eight; BACK: and above eight, so that a cut piece
// has its row's values before it.
//
// A team takes consecutive rows: what belongs to the channels is loaded once,
// before the first row (so that one row's call waits for memory once), and a
// gate row's activation is computed once for the rows that share it.
template <class T, int C, int BLOCK, bool TAIL, bool BACK>
__global__ __launch_bounds__(BLOCK) void residual_norm_kernel(Args p) {
  __shared__ Parts parts;
  const ResidualNormArgs& a = p.a;
  const int lane = threadIdx.x & 63, wb = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int W = p.W, w = wb & (W - 1), team = wb / W, teams = BLOCK / kWave / W, D = (int)a.D;
  const half_t *ax = (const half_t*)a.x, *ay = (const half_t*)a.y, *ag = (const half_t*)a.gate;
  int at[C], nv[C];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    at[j] = (j * W + w) * kPiece + lane * 8;
    const int left = D - at[j];
    nv[j] = left < 0 ? 0 : left > 8 ? 8 : left;
  }
  const int64_t first = ((int64_t)blockIdx.x * teams + team) * p.rows;
  const unsigned one = T::kOne * 0x10001u;
  u32x4 qg[C], qb[C], rg[C], rb[C];
  load_channels<C, BACK>(qg, (const half_t*)a.post_gamma, at, nv, one);
  load_channels<C, BACK>(qb, (const half_t*)a.post_beta, at, nv, 0);
  load_channels<C, BACK>(rg, (const half_t*)a.gamma, at, nv, one);
  load_channels<C, BACK>(rb, (const half_t*)a.beta, at, nv, 0);
  // the gate row in hand, and the first row that it no longer serves
  float g[C][8];
  int64_t grow = ag ? first / p.per : 0, gend = 0;
  // the whole workgroup walks the rows together: every wave takes every barrier
  for (int64_t i = 0; i < p.rows; ++i) {
    const bool live = first + i < a.M;
    const int64_t row = live ? first + i : a.M - 1, base = row * D;
    float v[C][8];
    if (ay) {
      u32x4 x[C], y[C];
#pragma unroll
      for (int j = 0; j < C; ++j) y[j] = load_raw8<BACK>(ay + base + at[j], nv[j]);
#pragma unroll
      for (int j = 0; j < C; ++j) x[j] = load_raw8<BACK>(ax + base + at[j], nv[j]);
      if (ag && live && row >= gend) {
        if (i) ++grow;
        gend = (grow + 1) * p.per;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          load8<T, BACK>(ag + grow * D + at[j], nv[j], g[j]);
          apply_act8(g[j], a.gate_act);
        }
      }
#pragma unroll
      for (int j = 0; j < C; ++j) widen8<T>(y[j], v[j]);
      if (a.post != GP_NORM_NONE) {
        float mean, rstd;
        row_stats<C, TAIL>(v, nv, a.post, D, W, w, a.post_eps, parts[i & 1][0], mean, rstd);
        affine<T, C>(v, mean, rstd, qg, qb, a.post_beta != nullptr);
      }
      if (ag) {
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] *= g[j][e];
      }
#pragma unroll
      for (int j = 0; j < C; ++j) {
        float f[8];
        widen8<T>(x[j], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float h = __builtin_fmaf(a.scale, v[j][e], f[e]);
          v[j][e] = (TAIL ? e < nv[j] : nv[j] > 0) ? h : 0.f;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) load8<T, BACK>(ax + base + at[j], nv[j], v[j]);
    }
    if (a.h && live) {
#pragma unroll
      for (int j = 0; j < C; ++j) store8<T>((half_t*)a.h + base + at[j], nv[j], v[j]);
    }
    // Pre takes h as it is in 32 bits, not as it was rounded into memory: out
    // has then one rounding, its own
    if (a.pre != GP_NORM_NONE) {
      float mean, rstd;
      row_stats<C, TAIL>(v, nv, a.pre, D, W, w, a.eps, parts[i & 1][1], mean, rstd);
      affine<T, C>(v, mean, rstd, rg, rb, a.beta != nullptr);
      if (live) {
#pragma unroll
        for (int j = 0; j < C; ++j) store8<T>((half_t*)a.out + base + at[j], nv[j], v[j]);
      }
    }
  }
}

template <class T, bool TAIL, bool BACK>
hipError_t launch(const Args& p, int C, int block, unsigned grid, hipStream_t s) {
#define GP_CASE(c, b)                                                                                  \
  if (C <= c && block == b) {                                                                          \
    hipLaunchKernelGGL((residual_norm_kernel<T, c, b, TAIL, BACK>), dim3(grid), dim3(b), 0, s, p);     \
    return hipGetLastError();                                                                          \
  }
  // rows above 16,384 values only have more than two pieces a wave
  GP_CASE(1, 256) GP_CASE(2, 256) GP_CASE(1, 512) GP_CASE(2, 512) GP_CASE(1, 1024) GP_CASE(2, 1024) GP_CASE(4, 1024)
#undef GP_CASE
  return hipErrorInvalidValue;
}

template <class T>
hipError_t by_tail(const Args& p, int C, int block, unsigned grid, hipStream_t s) {
  if (p.a.D % 8 == 0) return launch<T, false, false>(p, C, block, grid, s);
  if (p.a.D > 8) return launch<T, true, true>(p, C, block, grid, s);
  hipLaunchKernelGGL((residual_norm_kernel<T, 1, 256, true, false>), dim3(grid), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t residual_norm_launch(const ResidualNormArgs& a, int num_cus, hipStream_t s) {
  const int pieces = (int)((a.D + kPiece - 1) / kPiece);
  // Waves a row: two pieces each where rows are many (16,384 x 4,096: four waves
  // 103 us, eight 111, two 133; 16,288 x 1,021: one 47, two 47), one piece where
  // rows leave CUs without work (one row of 4,096: eight waves 3.6 us, four 4.3;
  // 128 rows of 8,192: sixteen 6.0, eight 6.8).
  int W = 1;
  while (W < kMaxWaves && pieces > 2 * W) W *= 2;
  if (a.M * W < 8 * num_cus)
    while (W < kMaxWaves && pieces > W) W *= 2;
  const int C = (pieces + W - 1) / W;
  const int block = W <= 4 ? 256 : W * kWave;
  const int64_t teams = block / kWave / W;
  // Up to four rows a team, so that what belongs to the channels is loaded once
  // for them, but not so many that workgroups get fewer than four a CU
  // (16,384 x 4,096: four rows 103 us, two 112, sixteen 125).  More where a
  // launch would pass the 2^32 - 1 threads that it may have.
  const int64_t groups = (a.M + teams - 1) / teams, most = (groups + 4 * num_cus - 1) / (4 * num_cus);
  const int64_t limit = ((int64_t(1) << 32) - 1) / block, least = (groups + limit - 1) / limit;
  const int64_t four = most < 4 ? most : 4, rows = four > least ? four : least;
  const int64_t grid = (a.M + teams * rows - 1) / (teams * rows);
  const Args p{a, W, rows, a.gate ? a.M / a.gate_rows : 1};
  return a.dtype == GP_DTYPE_BF16 ? by_tail<BF16>(p, C, block, (unsigned)grid, s)
                                  : by_tail<F16>(p, C, block, (unsigned)grid, s);
}

}  // namespace gp
