// Products with 4-bit weights: out = act(x W + b) [or x W + b + r], and the
// gated pair act(x Wg + bg) * (x Wu + bu), W[k][n] = s[k / G][n] (q[k][n] - z[k / G][n]).
// No counterpart in the reference, whose GEMM stages take 16-bit weights
// (common/bulksync_gemm.cuh:13-110).
//
// Words.  Word [k / 8][n] holds q of eight consecutive k, the lowest in the low
// bits: eight k of one column are what one lane of an MFMA holds, so a word is
// a lane's operand, and the weights need no other layout than [K / 8, N].
//
// From a word to an operand.  A 4-bit q in the top mantissa bits of 16.0 is the
// 16-bit float 16 + q, exactly, in fp16 and in bf16; one shift and one
// and-or make two of them, of k and k + 4, so the operand holds the eight k in
// the order 0 4 1 5 2 6 3 7, and x is put in the same order.  Per group of G
// rows the matrix cores sum x (16 + q) and, against a column of ones, x; then
//   sum x (q - z) = sum x (16 + q) - (16 + z) sum x
// in fp32, and times s into the running sum.  The weights are never rounded:
// what is lost is a few bits of fp32 where the two sums cancel.
#include <hip/hip_runtime.h>

#include "../../include/gpipes.h"
#include "gp_kernels.hpp"
#include "row_ops.hpp"

namespace gp {
namespace {

typedef unsigned short us4 __attribute__((ext_vector_type(4), aligned(2)));

template <class T>
struct Q4;
template <>
struct Q4<F16> : F16 {
  static constexpr int kShift = 6;  // q to the top of fp16's ten mantissa bits
  static constexpr unsigned kMask = 0x03C003C0u, kBase = 0x4C004C00u;
  __device__ static f4 mma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Q4<BF16> : BF16 {
  static constexpr int kShift = 3;  // of bf16's seven
  static constexpr unsigned kMask = 0x00780078u, kBase = 0x41804180u;
  __device__ static f4 mma16(h8 a, h8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  }
};

// The operand 16 + q of a word, k order 0 4 1 5 2 6 3 7.
template <class T>
__device__ __forceinline__ h8 q4_operand(unsigned w) {
  constexpr int s = Q4<T>::kShift;
  u32x4 o;
  o[0] = ((w << s) & Q4<T>::kMask) | Q4<T>::kBase;
  o[1] = ((s >= 4 ? w << (s - 4) : w >> (4 - s)) & Q4<T>::kMask) | Q4<T>::kBase;
  o[2] = ((w >> (8 - s)) & Q4<T>::kMask) | Q4<T>::kBase;
  o[3] = ((w >> (12 - s)) & Q4<T>::kMask) | Q4<T>::kBase;
  return __builtin_bit_cast(h8, o);
}

// Eight values of x in that order.
__device__ __forceinline__ h8 x_operand(u32x4 v) {
  u32x4 o;
  o[0] = __builtin_amdgcn_perm(v[2], v[0], 0x05040100u);
  o[1] = __builtin_amdgcn_perm(v[2], v[0], 0x07060302u);
  o[2] = __builtin_amdgcn_perm(v[3], v[1], 0x05040100u);
  o[3] = __builtin_amdgcn_perm(v[3], v[1], 0x07060302u);
  return __builtin_bit_cast(h8, o);
}

// The epilogue of one output: v the product (with two weights the gate's, and
// u the other's), in fp32 until it is stored.
template <class T>
__device__ __forceinline__ void q4_store(const Q4Args& p, int64_t m, int n, float v, float u) {
  if (p.side[0].b) v += T::val(((const half_t*)p.side[0].b)[n]);
  v = apply_act_ext(v, p.act);
  if (p.sides == 2) v *= p.side[1].b ? u + T::val(((const half_t*)p.side[1].b)[n]) : u;
  if (p.r) v += T::val(((const half_t*)p.r)[m * p.N + n]);
  ((half_t*)p.out)[m * p.N + n] = T::cvt1(v);
}

constexpr int kChunk = 128;  // k that a wave loads at a time: four MFMA steps, one to four groups

// ---------------------------------------------------------------------------
// Few rows: every wave of a workgroup multiplies its share of k with the
// workgroup's 16 CW columns, and the shares are joined through LDS in the
// order of the waves.  With two weights, half of the waves take each.
// ---------------------------------------------------------------------------
template <int CW, int MT, int SPC>
struct Chunk {
  unsigned w[4][CW];
  u32x4 x[4][MT];
  unsigned short s[SPC][CW], z[SPC][CW];
};

template <class T, int CW, int MT, int G, bool FOUR>
__global__ __launch_bounds__(MT == 1 ? 1024 : 512) void q4_rows_kernel(Q4Args p) {
  constexpr int SPC = kChunk / G;        // groups a chunk
  constexpr int SPG = G / 32;            // MFMA steps a group
  constexpr int E = FOUR ? 1 : 4;        // accumulator elements that hold rows (FOUR: at most four rows)
  constexpr int COLS = 16 * CW;
  constexpr int TOK = FOUR ? 4 : 16;
  __shared__ float part[(MT == 1 ? 16 : 8) * TOK * COLS];
  const int lane = threadIdx.x & 63, j = lane & 15, lg = lane >> 4;
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = waves / p.sides;  // waves a weight
  const int side = wave / per, wk = wave - side * per;
  const int N = p.N, K = p.K;
  const int n0 = blockIdx.x * COLS;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const int rows = p.M - m0 < 16 * MT ? (int)(p.M - m0) : 16 * MT;
  const int groups = (K + G - 1) / G;
  const int chunks = (K + kChunk - 1) / kChunk;
  const Q4Side sd = side ? p.side[1] : p.side[0];
  const auto wr = make_rsrc(sd.wq, (int)((int64_t)K * N / 2));
  const auto xr = make_rsrc((const half_t*)p.x + m0 * K, rows * K * 2);
  const unsigned short* sp = (const unsigned short*)sd.s;
  const unsigned short* zp = (const unsigned short*)sd.z;
  const int col = n0 + CW * j;
  const bool inside = n0 + COLS <= N;
  // Row i of the x operand: row i, or with at most four rows row i / 4, which
  // lands in element 0 of the accumulators of the lanes of group i / 4.
  const int xrow = FOUR ? j >> 2 : j;

  auto load = [&](int c, Chunk<CW, MT, SPC>& q) {
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      const int k8 = c * (kChunk / 8) + st * 4 + lg;
      const int off = (int)(((unsigned)k8 * (unsigned)N + (unsigned)col) * 4u);  // past the weight's end: zeros
      if constexpr (CW == 4) {
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(wr, off, 0, 0);
        for (int t = 0; t < 4; ++t) q.w[st][t] = v[t];
      } else if constexpr (CW == 2) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(wr, off, 0, 0);
        q.w[st][0] = v[0], q.w[st][1] = v[1];
      } else {
        q.w[st][0] = __builtin_amdgcn_raw_buffer_load_b32(wr, off, 0, 0);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        // past the row's end (and past the last row) nothing is read: zeros, which no word can make count
        const int xo = ((mt * 16 + xrow) * K + k8 * 8) * 2;
        q.x[st][mt] = __builtin_amdgcn_raw_buffer_load_b128(xr, k8 * 8 < K ? xo : 0x7FFFFFF0, 0, 0);
      }
    }
#pragma unroll
    for (int g = 0; g < SPC; ++g) {
      const int gi = c * SPC + g < groups ? c * SPC + g : groups - 1;
      const int64_t at = (int64_t)gi * N;
#pragma unroll
      for (int t = 0; t < CW; ++t) {
        const int cc = inside || col + t < N ? col + t : N - 1;
        q.s[g][t] = sp[at + cc];
        q.z[g][t] = zp ? zp[at + cc] : 0;
      }
    }
  };

  float tot[CW][MT][E] = {};
  const h8 ones = __builtin_bit_cast(h8, u32x4{T::kOne * 0x10001u, T::kOne * 0x10001u, T::kOne * 0x10001u,
                                               T::kOne * 0x10001u});
  auto mul = [&](const Chunk<CW, MT, SPC>& q) {
#pragma unroll
    for (int g = 0; g < SPC; ++g) {
      f4 acc[CW][MT] = {}, sum[MT] = {};
#pragma unroll
      for (int st = g * SPG; st < (g + 1) * SPG; ++st) {
        h8 b[CW];
#pragma unroll
        for (int t = 0; t < CW; ++t) b[t] = q4_operand<T>(q.w[st][t]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const h8 a = x_operand(q.x[st][mt]);
          sum[mt] = Q4<T>::mma16(a, ones, sum[mt]);
#pragma unroll
          for (int t = 0; t < CW; ++t) acc[t][mt] = Q4<T>::mma16(a, b[t], acc[t][mt]);
        }
      }
#pragma unroll
      for (int t = 0; t < CW; ++t) {
        const float s = T::val(__builtin_bit_cast(half_t, q.s[g][t]));
        const float z = zp ? 16.f + T::val(__builtin_bit_cast(half_t, q.z[g][t])) : 24.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < E; ++e)
            tot[t][mt][e] = __builtin_fmaf(s, __builtin_fmaf(-z, sum[mt][e], acc[t][mt][e]), tot[t][mt][e]);
      }
    }
  };

  // wave wk of the weight's `per` takes chunks wk, wk + per, ..., the next one's loads under this one's products
  Chunk<CW, MT, SPC> qa, qb;
  int c = wk;
  if (c < chunks) load(c, qa);
  while (c < chunks) {
    if (c + per < chunks) load(c + per, qb);
    mul(qa);
    if ((c += per) >= chunks) break;
    if (c + per < chunks) load(c + per, qa);
    mul(qb);
    c += per;
  }

#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (mt) __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int t = 0; t < CW; ++t)
        part[(wave * TOK + (FOUR ? lg : 4 * lg + e)) * COLS + CW * j + t] = tot[t][mt][e];
    __syncthreads();
    for (int i = threadIdx.x; i < TOK * COLS; i += blockDim.x) {
      const int row = mt * 16 + i / COLS, n = n0 + i % COLS;
      if (row >= rows || n >= N) continue;
      float v = 0.f, u = 0.f;
      for (int w = 0; w < per; ++w) v += part[w * TOK * COLS + i];
      for (int w = per; w < waves; ++w) u += part[w * TOK * COLS + i];
      q4_store<T>(p, m0 + row, n, v, u);
    }
  }
}

template <class T, int CW, int MT, bool FOUR>
hipError_t rows_launch(const Q4Args& a, int waves, dim3 grid, hipStream_t s) {
  const dim3 block(waves * kWave);
  switch (a.group) {
    case 32: hipLaunchKernelGGL((q4_rows_kernel<T, CW, MT, 32, FOUR>), grid, block, 0, s, a); break;
    case 64: hipLaunchKernelGGL((q4_rows_kernel<T, CW, MT, 64, FOUR>), grid, block, 0, s, a); break;
    case 128: hipLaunchKernelGGL((q4_rows_kernel<T, CW, MT, 128, FOUR>), grid, block, 0, s, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

template <class T>
hipError_t launch(const Q4Args& a, int num_cus, hipStream_t s) {
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
  int waves = mt == 1 ? 16 : 8;
  while (waves > 2 * a.sides && waves / 2 >= chunks * a.sides) waves /= 2;
  const int cw = a.N >= 64 * num_cus ? 4 : a.N >= 32 * num_cus ? 2 : 1;
  const dim3 grid((unsigned)((a.N + 16 * cw - 1) / (16 * cw)), (unsigned)((a.M + 16 * mt - 1) / (16 * mt)));
#define GP_CASE(c, m, four) \
  if (cw == c && mt == m && (a.M <= 4) == four) return rows_launch<T, c, m, four>(a, waves, grid, s);
  GP_CASE(1, 1, true) GP_CASE(2, 1, true) GP_CASE(4, 1, true)
  GP_CASE(1, 1, false) GP_CASE(2, 1, false) GP_CASE(4, 1, false)
  GP_CASE(1, 2, false) GP_CASE(2, 2, false) GP_CASE(4, 2, false)
  GP_CASE(1, 4, false) GP_CASE(2, 4, false) GP_CASE(4, 4, false)
#undef GP_CASE
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t q4_launch(const Q4Args& a, int num_cus, hipStream_t s) {
  return a.dtype == GP_DTYPE_BF16 ? launch<BF16>(a, num_cus, s) : launch<F16>(a, num_cus, s);
}

}  // namespace gp
