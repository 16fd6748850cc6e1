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
// its load to its store, and every statistic is taken from there.
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
// statistics are in 32 bits throughout.
template <int C>
__device__ __forceinline__ void row_stats(const float (&v)[C][8], const int (&nv)[C], int kind, int64_t D, int W, int w,
                                          float eps, Part* parts, float& mean, float& rstd) {
  Part p{0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int64_t left = D - (int64_t)(j * W + w) * kPiece;
    p.n += (float)(left < 0 ? 0 : left > kPiece ? kPiece : left);
  }
  if (kind == GP_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[j][e];  // values past the row's end are zeros
    p.mean = p.n > 0.f ? sum_lanes<64>(s) / p.n : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < C; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = e < nv[j] ? v[j][e] - p.mean : 0.f;
      q = __builtin_fmaf(d, d, q);
    }
  p.m2 = sum_lanes<64>(q);
  if (W > 1) {
    const int lane = threadIdx.x & 63, wb = threadIdx.x >> 6;
    if (lane == 0) parts[wb] = p;
    __syncthreads();
    const int i = lane & 15;
    p = Part{0.f, 0.f, 0.f};
    if (i < W) p = parts[wb - w + i];
    const float m = sum_lanes<16>(p.n * p.mean) / (float)D;
    p.m2 = sum_lanes<16>(__builtin_fmaf(p.n * (p.mean - m), p.mean - m, p.m2));
    p.mean = m;
  }
  mean = p.mean;
  // a precise division and root: once a row, and rsq's last bit would scale every value
  rstd = 1.f / __builtin_sqrtf(p.m2 / (float)D + eps);
}

struct Args {
  ResidualNormArgs a;
  int W;          // waves a row
  int64_t per;    // rows that share a gate row
};

// (v - mean) rstd gamma + beta over this thread's values.
template <class T, int C>
__device__ __forceinline__ void affine(float (&v)[C][8], const int (&nv)[C], const int (&at)[C], float mean, float rstd,
                                       const void* gamma, const void* beta) {
#pragma unroll
  for (int j = 0; j < C; ++j) {
    float g[8], b[8];
    if (gamma) load8<T>((const half_t*)gamma + at[j], nv[j], g);
    if (beta) load8<T>((const half_t*)beta + at[j], nv[j], b);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float u = (v[j][e] - mean) * rstd;
      u = __builtin_fmaf(u, gamma ? g[e] : 1.f, beta ? b[e] : 0.f);
      v[j][e] = e < nv[j] ? u : 0.f;
    }
  }
}

template <class T, int C, int BLOCK>
__global__ __launch_bounds__(BLOCK) void residual_norm_kernel(Args p) {
  __shared__ Parts parts;
  const ResidualNormArgs& a = p.a;
  const int lane = threadIdx.x & 63, wb = threadIdx.x >> 6;
  const int W = p.W, w = wb % W, team = wb / W, teams = BLOCK / kWave / W;
  int at[C], nv[C];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    at[j] = (j * W + w) * kPiece + lane * 8;
    const int64_t left = a.D - at[j];
    nv[j] = left < 0 ? 0 : left > 8 ? 8 : (int)left;
  }
  int par = 0;
  // the whole workgroup walks the rows together: every wave takes every barrier
  for (int64_t r0 = (int64_t)blockIdx.x * teams; r0 < a.M; r0 += (int64_t)gridDim.x * teams, par ^= 1) {
    const int64_t row = r0 + team;
    const bool live = row < a.M;
    const int64_t base = (live ? row : a.M - 1) * a.D;
    float v[C][8];
    if (a.y) {
      float x[C][8];
#pragma unroll
      for (int j = 0; j < C; ++j) load8<T>((const half_t*)a.y + base + at[j], nv[j], v[j]);
#pragma unroll
      for (int j = 0; j < C; ++j) load8<T>((const half_t*)a.x + base + at[j], nv[j], x[j]);
      if (a.post != GP_NORM_NONE) {
        float mean, rstd;
        row_stats<C>(v, nv, a.post, a.D, W, w, a.post_eps, parts[par][0], mean, rstd);
        affine<T, C>(v, nv, at, mean, rstd, a.post_gamma, a.post_beta);
      }
      if (a.gate) {
        const int64_t gb = (live ? row : a.M - 1) / p.per * a.D;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          float g[8];
          load8<T>((const half_t*)a.gate + gb + at[j], nv[j], g);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] *= apply_act_ext(g[e], a.gate_act);
        }
      }
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = e < nv[j] ? __builtin_fmaf(a.scale, v[j][e], x[j][e]) : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) load8<T>((const half_t*)a.x + base + at[j], nv[j], v[j]);
    }
    if (a.h && live) {
#pragma unroll
      for (int j = 0; j < C; ++j) store8<T>((half_t*)a.h + base + at[j], nv[j], v[j]);
    }
    // Pre takes h as it is in 32 bits, not as it was rounded into memory: out
    // has then one rounding, its own
    if (a.pre != GP_NORM_NONE) {
      float mean, rstd;
      row_stats<C>(v, nv, a.pre, a.D, W, w, a.eps, parts[par][1], mean, rstd);
      affine<T, C>(v, nv, at, mean, rstd, a.gamma, a.beta);
      if (live) {
#pragma unroll
        for (int j = 0; j < C; ++j) store8<T>((half_t*)a.out + base + at[j], nv[j], v[j]);
      }
    }
  }
}

template <class T>
hipError_t launch(const Args& p, int C, int block, unsigned grid, hipStream_t s) {
#define GP_CASE(c, b)                                                                                \
  if (C <= c && block == b) {                                                                        \
    hipLaunchKernelGGL((residual_norm_kernel<T, c, b>), dim3(grid), dim3(b), 0, s, p);               \
    return hipGetLastError();                                                                        \
  }
  GP_CASE(1, 256) GP_CASE(2, 256) GP_CASE(4, 256)
  GP_CASE(1, 512) GP_CASE(2, 512) GP_CASE(4, 512)
  GP_CASE(1, 1024) GP_CASE(2, 1024) GP_CASE(4, 1024)
#undef GP_CASE
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t residual_norm_launch(const ResidualNormArgs& a, int num_cus, hipStream_t s) {
  const int pieces = (int)((a.D + kPiece - 1) / kPiece);
  int W = 1;
  while (W < kMaxWaves && pieces > 4 * W) W *= 2;
  const int C = (pieces + W - 1) / W;
  const int block = W <= 4 ? 256 : W * kWave;
  const int64_t teams = block / kWave / W;
  const int64_t groups = (a.M + teams - 1) / teams;
  const int64_t most = (int64_t)num_cus * (2048 / block);
  const Args p{a, W, a.gate ? a.M / a.gate_rows : 1};
  const unsigned grid = (unsigned)(groups < most ? groups : most);
  return a.dtype == GP_DTYPE_BF16 ? launch<BF16>(p, C, block, grid, s) : launch<F16>(p, C, block, grid, s);
}

}  // namespace gp
