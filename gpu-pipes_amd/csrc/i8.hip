// Products in 8-bit integers with a scale for each row of x and each column of
// the weight: out = act(x W + b) [or x W + b + r], and the gated pair
// act(x Wg + bg) * (x Wu + bu).  No counterpart in the reference, whose GEMM
// stages take 16-bit operands (common/bulksync_gemm.cuh:13-110).
//
//   q[m][k] = rint(127 x[m][k] / a[m]), a[m] = max |x[m][.]|, xs[m] = a[m] / 127
//   (x W)[m][n] = xs[m] ws[n] sum_k q[m][k] wq[k][n]
//
// The sums are exact: whole numbers in 32 bits, K at most 131,056.  So neither
// the order of k nor the number of parts it is cut into changes a result, and
// a row's bits are the same from every kernel here.
//
// Weights.  Blocks of 16 columns by 64 k, 1 KiB: byte 256 g + 16 j + i of block
// [n / 16][k / 64] is wq[64 (k / 64) + 16 g + i][16 (n / 16) + j], the operand
// of a 16 x 16 x 64 MFMA as its lanes hold it (lane 16 g + j).  Blocks of a
// column tile follow each other along k, so a wave streams whole lines and an
// operand's read from LDS is 1 KiB in a row.  Behind K and N the blocks hold
// zeros, and a zero times whatever integer lies behind a row of x is zero: rows
// of x need no padding.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/gpipes.h"
#include "gp_kernels.hpp"
#include "row_ops.hpp"

// No sum is fused with a product that the source does not fuse: what one kernel rounds, every kernel rounds.
#pragma clang fp contract(off)

namespace gp {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int i4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kChunk = 128;  // k that a wave or a workgroup takes at a time: a line of a row of x
constexpr unsigned kNowhere = 0xFFFFFFE0u;  // a buffer offset past every end: reads bring zeros

__device__ __forceinline__ i32x4 mma8(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// Workgroup b of n, renumbered so that neighbours in the result run on one XCD (b % 8).
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int x = b & 7, i = b >> 3, q = n >> 3, rem = n & 7;
  return x * q + (x < rem ? x : rem) + i;
}

// ---------------------------------------------------------------------------
// A row's whole numbers.  With x and a scaled by one power of two, 127 x is
// exact in fp32 (18 bits) and so is the remainder 127 x - q a; the quotient,
// corrected once by its remainder, is the correctly rounded one.  A quotient
// of 11-bit numbers that is not itself halfway between two whole numbers is
// further from every half than 32 times what it can be off by, so its rounding
// (ties to even) is that of the exact quotient.
// ---------------------------------------------------------------------------
struct RowScale {
  float up;     // the power of two
  float top;    // a * up
  float inv;    // 1 / top, or 0 for a row of zeros and one that is not finite
  float scale;  // xs
};

// bits: the largest |x| of the row as the element type's bits (an infinity or NaN is larger than any number).
template <class T>
__device__ __forceinline__ RowScale row_scale(unsigned bits) {
  const float a = T::val(__builtin_bit_cast(half_t, (unsigned short)bits));
  int e = 254 - (int)(__builtin_bit_cast(unsigned, a) >> 23);
  e = e < 1 ? 1 : e > 247 ? 247 : e;  // 127 * up stays finite
  RowScale s;
  s.up = __builtin_bit_cast(float, (unsigned)e << 23);
  s.top = a * s.up;
  const bool finite = a < __builtin_inff();
  s.inv = finite && a > 0.f ? 1.f / s.top : 0.f;
  s.scale = finite ? a / 127.f : __builtin_nanf("");
  return s;
}

// Four values as bytes.  Adding 1.5 * 2^23 rounds to a whole number, which then stands in the low bits.
__device__ __forceinline__ unsigned round4(const float* x, const RowScale& s) {
  unsigned u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = x[i] * (127.f * s.up);
    float q = t * s.inv;
    q = __builtin_fmaf(__builtin_fmaf(-q, s.top, t), s.inv, q);
    u[i] = __builtin_bit_cast(unsigned, q + 12582912.f);
  }
  const unsigned lo = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000C0Cu);
  return s.inv == 0.f ? 0u : lo | hi;  // an infinity times 0 has no whole number
}
template <class T>
__device__ __forceinline__ u32x2 round8(u32x4 v, const RowScale& s) {
  float f[8];
  widen8<T>(v, f);
  return u32x2{round4(f, s), round4(f + 4, s)};
}

// Larger of the 15-bit magnitudes in both halves.
__device__ __forceinline__ unsigned top2(unsigned a, unsigned v) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  const u16x2 m = __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, v & 0x7FFF7FFFu));
  return __builtin_bit_cast(unsigned, m);
}
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
// The largest half over the wave, in every lane.
__device__ __forceinline__ unsigned wave_top(unsigned a) {
  unsigned m = umax(a & 0xFFFF, a >> 16);
#define GP_DPP(v, ctrl) (unsigned)__builtin_amdgcn_mov_dpp((int)(v), ctrl, 0xF, 0xF, false)
  m = umax(m, GP_DPP(m, 0x128));  // row_ror:8
  m = umax(m, GP_DPP(m, 0x124));
  m = umax(m, GP_DPP(m, 0x4E));
  m = umax(m, GP_DPP(m, 0xB1));
#undef GP_DPP
  auto p = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  m = umax(p[0], p[1]);
  p = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return umax(p[0], p[1]);
}

// Rows of x to bytes: WPR waves a row, P pieces of eight values a lane held in
// registers, so that memory is read once; rows longer than that are read again
// (from L2).  One wave a row up to 2,048 values.  block: of WAVES / WPR rows.
// count: where it is given, the rows that there are.  part: one value a wave.
template <class T, int P, int WPR, int WAVES>
__device__ __forceinline__ void rows_to_bytes(const half_t* x, int64_t M, int K, char* q, float* xs, const int* count,
                                              int64_t block, unsigned* part) {
  constexpr int STEP = 64 * WPR * 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = wave / WPR * WPR;
  int64_t m = block * (WAVES / WPR) + wave / WPR;
  const bool in = m < M && !(count && m >= *count);
  m = in ? m : 0;  // such a wave reads nothing, but comes to the barrier
  const auto xr = make_rsrc(x + m * K, in ? K * 2 : 0);
  const int at = (lane + (wave - first) * 64) * 8;
  u32x4 v[P];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, (at + i * STEP) * 2, 0, 0);
#pragma unroll
  for (int i = 0; i < P; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = top2(top, v[i][e]);
  for (int k = at + P * STEP; k < K; k += STEP) {
    const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(xr, k * 2, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) top = top2(top, w[e]);
  }
  top = wave_top(top);
  if constexpr (WPR > 1) {
    if (lane == 0) part[wave] = top;
    __syncthreads();
    top = wave_top(part[first + (lane & (WPR - 1))]);
  }
  if (!in) return;
  const RowScale s = row_scale<T>(top);
  char* const row = q + m * K;
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (at + i * STEP < K) *(u32x2*)(row + at + i * STEP) = round8<T>(v[i], s);
  for (int k = at + P * STEP; k < K; k += STEP)
    *(u32x2*)(row + k) = round8<T>(__builtin_amdgcn_raw_buffer_load_b128(xr, k * 2, 0, 0), s);
  if (at == 0) xs[m] = s.scale;
}
template <class T, int P, int WPR, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void i8_rows_to_bytes_kernel(const half_t* x, int64_t M, int K, char* q, float* xs,
                                                                     const int* count) {
  __shared__ unsigned part[WAVES];
  rows_to_bytes<T, P, WPR, WAVES>(x, M, K, q, xs, count, (int64_t)blockIdx.y * gridDim.x + blockIdx.x, part);
}

template <class T>
hipError_t rows_to_bytes_launch(const void* x, int64_t M, int K, char* q, float* xs, hipStream_t s, const int* count = nullptr) {
  const half_t* h = (const half_t*)x;
  // a launch holds fewer than 2^32 threads along an axis, and experts have up to 2^26 rows
  auto grid = [&](int rows) {
    const int64_t n = (M + rows - 1) / rows, most = 1 << 20, y = (n + most - 1) / most;
    return dim3((unsigned)((n + y - 1) / y), (unsigned)y);
  };
#define GP_ROWS(p, w, waves)                                                                                        \
  hipLaunchKernelGGL((i8_rows_to_bytes_kernel<T, p, w, waves>), grid(waves / w), dim3(64 * waves), 0, s, h, M, K, q, \
                     xs, count)
  if (K <= 512) GP_ROWS(1, 1, 4);
  else if (K <= 2048) GP_ROWS(4, 1, 4);
  else if (K <= 8192) GP_ROWS(4, 4, 4);
  else GP_ROWS(4, 16, 16);
#undef GP_ROWS
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Epilogue
// ---------------------------------------------------------------------------
// The stages' activations and SiLU; a NaN stays one under every one of them.
__device__ __forceinline__ float act8(float v, int act) { return act == GP_ACT_RELU ? (v < 0.f ? 0.f : v) : apply_act_ext(v, act); }

// The first cnt of eight values from column n of a row of N, zeros behind them.
// Loads under a condition each are waited for one by one, so a row's end is read
// with what lies before it (and a scale with zeros behind N, by the buffer's range).
template <class T>
__device__ __forceinline__ void load_row8(const half_t* row, int n, int cnt, int N, float (&f)[8]) {
  if (N >= 8)
    load8<T, true>(row + n, cnt, f);
  else
    load8<T>(row + n, cnt, f);
}
__device__ __forceinline__ void load_scales8(const float* s, int n, int N, float (&f)[8]) {
  const auto r = make_rsrc(s, N * 4);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f4 v = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(r, (n + 4 * h) * 4, 0, 0));
#pragma unroll
    for (int e = 0; e < 4; ++e) f[4 * h + e] = v[e];
  }
}

// cnt of eight neighbouring outputs of a row from column n: v (and u of the second
// weight) the sums times both scales, b the biases, zeros where there are none
// (BIAS false: of a product that has none).
template <class T, int S, bool BIAS = true>
__device__ __forceinline__ void finish8(const I8Args& p, int64_t m, int n, int cnt, float (&v)[8], float (&u)[8],
                                        const float (&b)[S][8]) {
  if constexpr (BIAS) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += b[0][e];
  }
  if (p.act == GP_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
  } else {
    apply_act8(v, p.act);
  }
  if constexpr (S == 2) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= BIAS ? u[e] + b[1][e] : u[e];
  }
  if (p.r) {
    float t[8];
    load_row8<T>((const half_t*)p.r + m * p.N, n, cnt, p.N, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
  }
  store8<T>((half_t*)p.out + m * p.N + n, cnt, v);
}

// One output.
template <class T, int S>
__device__ __forceinline__ void finish1(const I8Args& p, int64_t m, int n, float v, float u) {
  v += p.side[0].b ? T::val(((const half_t*)p.side[0].b)[n]) : 0.f;
  v = act8(v, p.act);
  if constexpr (S == 2) v *= u + (p.side[1].b ? T::val(((const half_t*)p.side[1].b)[n]) : 0.f);
  if (p.r) v += T::val(((const half_t*)p.r)[m * p.N + n]);
  ((half_t*)p.out)[m * p.N + n] = T::cvt1(v);
}

// ---------------------------------------------------------------------------
// Experts: a product's rows lie in runs, one an expert, each cut into tiles.
// UP: tile rows are tokens of x, gathered, the results one after the other;
// DOWN: the rows one after the other, the results in fp32 at their (token,
// choice) pairs.
// ---------------------------------------------------------------------------
enum { DENSE, UP, DOWN };
struct TileRec {
  int expert, row0, rows, pad;
};
struct I8Group {
  const TileRec* tiles;
  const int* info;  // tiles and rows that there are
  const int* tok;   // of a row: its token
  const int* pair;  // and its pair, token * topk + choice
  int64_t wbytes;   // of an expert's packed weight
  int shift;        // a tile of the plan is 2^shift of the product's
  // Few tokens: every pair a tile by itself, without a plan.
  const int* ids;
  int topk, experts;
};

// ---------------------------------------------------------------------------
// Few rows.  A wave multiplies its share of k with NT tiles of 16 columns (of
// two weights NT / 2 of each); words and x go through a ring of R chunks in
// LDS that is the wave's own, so that many loads are in flight and no barrier
// lies between them, and the waves' sums are joined through LDS.
// XL: at most four rows of 16-bit x (own_bytes), which the workgroup makes bytes of itself.
// Bound by the weights' loads: a token's 2 x 16,384 columns from 4,096 k 27.8 us
// (134 MB, 4.8 TB/s), 4,096 from 16,384 k 11.7 to 13.3; 16 rows of 8,192 from 8,192 12.1.
// ---------------------------------------------------------------------------
constexpr int rows_ring(int nt, int mt, bool xl) { return xl ? 2 : nt + mt <= 3 ? 3 : 2; }
constexpr int slot_bytes(int nt, int mt, bool xl) { return (nt + (xl ? 0 : mt)) * 2048; }
constexpr int kRowsLds = 156 * 1024;  // of dynamic LDS at most
// Waves of a workgroup at most, a power of two: sixteen, or as many as have room for their rings.
constexpr int rows_waves(int nt, int mt, bool xl) {
  const int fit = (kRowsLds - (xl ? 20 * 1024 : 0)) / (rows_ring(nt, mt, xl) * slot_bytes(nt, mt, xl));
  return fit >= 16 ? 16 : fit >= 8 ? 8 : 4;
}

struct RowsPlan {
  int nt, mt, kw, cg;  // column tiles a wave, row tiles, waves along k, waves along the columns
  bool xl;
  int xstride, bytes;  // XL: of a row's bytes; LDS
};

template <class T, int S, int NT, int MT, bool XL, int MODE>
__global__ __launch_bounds__(64 * rows_waves(NT, MT, XL)) void i8_rows_kernel(I8Args p, I8Group grp, int kwshift,
                                                                             int mshift, int xstride) {
  constexpr int R = rows_ring(NT, MT, XL), SLOT = slot_bytes(NT, MT, XL), NI = SLOT / 1024, CW = NT / S;
  __shared__ unsigned tops[16];
  __shared__ float rowscale[16 * MT];
  __shared__ int rowpair[MODE == DOWN ? 16 * MT : 1];
  GP_LDS char* lds = dyn_lds();
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, lg = lane >> 4;
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KW = 1 << kwshift, kw = wave & (KW - 1), cg = wave >> kwshift, CG = waves >> kwshift;
  const int N = p.N, K = p.K, N16 = (N + 15) / 16, K64 = (K + 63) / 64, chunks = (K + kChunk - 1) / kChunk;
  const int t0 = xcd_order(blockIdx.x, gridDim.x) * (CW * CG);  // the workgroup's first tile of columns
  int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  int rows = p.M - m0 < 16 * MT ? (int)(p.M - m0) : 16 * MT;
  if constexpr (MODE != DENSE) {
    TileRec rec{0, (int)blockIdx.y, 1, 0};
    if constexpr (XL) {  // a pair; its token's row is the first of p.x
      rec.expert = grp.ids[blockIdx.y];
      if ((unsigned)rec.expert >= (unsigned)grp.experts) return;
      p.x = (const half_t*)p.x + (int64_t)(blockIdx.y / grp.topk) * K;
      p.M = 1;
    } else {
      if ((int)blockIdx.y >= grp.info[0]) return;
      rec = grp.tiles[blockIdx.y];
    }
    m0 = rec.row0, rows = rec.rows;
#pragma unroll
    for (int s = 0; s < S; ++s)
      p.side[s].wq = (const char*)p.side[s].wq + rec.expert * grp.wbytes, p.side[s].s += (int64_t)rec.expert * N;
  }

  // 16-bit x first: what follows is not waited for with it
  constexpr int XP = 4;
  u32x4 xv[XL ? XP : 1];
  const int tpr = blockDim.x >> mshift, xrow = XL ? tid / tpr : 0, xat = XL ? (tid - xrow * tpr) * 8 : 0;
  if constexpr (XL) {
    const auto xr = make_rsrc(p.x, (int)p.M * K * 2);
#pragma unroll
    for (int i = 0; i < XP; ++i) {
      const int k = xat + i * tpr * 8;
      xv[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, k < K ? (xrow * K + k) * 2 : (int)kNowhere, 0, 0);
    }
  }

  GP_LDS char* const ring = lds + wave * (R * SLOT);
  const int wbytes = N16 * K64 * 1024;
  const auto wr0 = make_rsrc(p.side[0].wq, wbytes);
  const auto wr1 = make_rsrc(p.side[S - 1].wq, wbytes);
  const auto xr8 = MODE == UP ? make_rsrc(p.xq, (int)(p.M * K)) : make_rsrc((const char*)p.xq + m0 * K, rows * K);
  unsigned wo[CW];
#pragma unroll
  for (int t = 0; t < CW; ++t) {
    const int n16 = t0 + cg * CW + t;
    wo[t] = n16 < N16 ? (unsigned)(n16 * K64) * 1024u + (unsigned)lane * 16u : 0xC0000000u;
  }
  // 16-byte piece c of row r lies at c ^ (r / 2) % 8: sixteen rows' reads of one piece fall into different banks
  const int dr = lane >> 3;
  unsigned xo[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = mt * 16 + 8 * h + dr;
      const unsigned piece = (unsigned)(((lane & 7) ^ ((row >> 1) & 7)) << 4);
      int from = row;
      if constexpr (MODE == UP && !XL)
        from = (int)__builtin_amdgcn_raw_buffer_load_b32(make_rsrc(grp.tok + m0, rows * 4), row * 4, 0, 0);
      xo[mt][h] = (unsigned)from * (unsigned)K + piece;
      if (MODE == UP && row >= rows) xo[mt][h] = 0x80000000u;
    }
  // What the epilogue needs of each row, asked for before the ring so as not to be waited for behind it.
  float rs = 0.f;
  int rp = 0;
  if (!XL && tid < rows) {
    rs = p.xs[MODE == UP ? grp.tok[m0 + tid] : m0 + tid];
    if (MODE == DOWN) rp = grp.pair[m0 + tid];
  }

  auto issue = [&](int c, int slot) {
    GP_LDS char* at = ring + slot * SLOT;
    const bool in = c < chunks;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int t = 0; t < CW; ++t)
#pragma unroll
        for (int b = 0; b < 2; ++b)
          dma16_buf(s ? wr1 : wr0, (int)(in && 2 * c + b < K64 ? wo[t] + (unsigned)(2 * c + b) * 1024u : kNowhere),
                    at + (s * CW + t) * 2048 + b * 1024);
    if constexpr (!XL) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          dma16_buf(xr8, (int)(in ? xo[mt][h] + (unsigned)(c * kChunk) : kNowhere),
                    at + NT * 2048 + mt * 2048 + h * 1024);
    }
  };
#pragma unroll
  for (int i = 0; i < R; ++i) issue(kw + i * KW, i);
  if (!XL && tid < rows) {
    rowscale[tid] = rs;
    if (MODE == DOWN) rowpair[tid] = rp;
  }

  GP_LDS char* const xl = lds + waves * (R * SLOT);
  if constexpr (XL) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < XP; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = top2(top, xv[i][e]);
    top = wave_top(top);
    if (lane == 0) tops[wave] = top;
    lds_barrier();
    const int wpr = waves >> mshift;
    top = wave_top(tops[xrow * wpr + (lane & (wpr - 1))]);
    const RowScale s = row_scale<T>(top);
#pragma unroll
    for (int i = 0; i < XP; ++i) {
      const int k = xat + i * tpr * 8;
      if (k < K) *(GP_LDS u32x2*)(xl + xrow * xstride + k) = round8<T>(xv[i], s);
    }
    if (xat == 0) rowscale[xrow] = s.scale;
    lds_barrier();
  }

  i32x4 acc[NT][MT] = {};
  const int nc = kw < chunks ? (chunks - 1 - kw) / KW + 1 : 0;
  const int sw = (j >> 1) & 7;
  int at = 0;
  for (int t = 0; t < nc; ++t) {
    const int c = kw + t * KW;
    wait_vmcnt<(R - 1) * NI>();
    compiler_fence();
    GP_LDS char* slot = ring + at * SLOT;
    u32x4 b[2][NT], a[2][MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < NT; ++n) b[h][n] = *(GP_LDS const u32x4*)(slot + n * 2048 + h * 1024 + lane * 16);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if constexpr (XL)
          a[h][mt] = *(GP_LDS const u32x4*)(xl + (j & ((1 << mshift) - 1)) * xstride + c * kChunk + h * 64 + lg * 16);
        else
          a[h][mt] = *(GP_LDS const u32x4*)(slot + NT * 2048 + mt * 2048 + j * 128 + (((4 * h + lg) ^ sw) << 4));
      }
    }
    // what was read is in registers before the slot takes the chunk R further on
    compiler_fence();
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    issue(c + R * KW, at);
    at = at + 1 == R ? 0 : at + 1;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[n][mt] = mma8(a[h][mt], b[h][n], acc[n][mt]);
  }

  // The waves' sums: wave (cg, kw) leaves rows of 16 NT in its own part of the ring.
  wait_vmcnt<0>();
  compiler_fence();
  constexpr int LD = 16 * NT;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) *(GP_LDS int*)(ring + ((mt * 16 + 4 * lg + e) * LD + n * 16 + j) * 4) = acc[n][mt][e];
  __syncthreads();
  const int cols = 16 * CW * CG;
  for (int i = tid; i < rows * cols; i += blockDim.x) {
    const int m = i / cols, c = i - m * cols, g = c / (16 * CW), n = t0 * 16 + c;
    if (n >= N) continue;
    GP_LDS const char* from = lds + (g << kwshift) * (R * SLOT) + (m * LD + (c - g * 16 * CW)) * 4;
    int v = 0, u = 0;
    for (int w = 0; w < KW; ++w) {
      v += *(GP_LDS const int*)(from + w * (R * SLOT));
      if (S == 2) u += *(GP_LDS const int*)(from + w * (R * SLOT) + 16 * CW * 4);
    }
    const float xsc = rowscale[m];
    if constexpr (MODE == DOWN)
      ((float*)p.out)[(int64_t)rowpair[m] * N + n] = (float)v * p.side[0].s[n] * xsc;
    else
      finish1<T, S>(p, m0 + m, n, (float)v * p.side[0].s[n] * xsc, S == 2 ? (float)u * p.side[S - 1].s[n] * xsc : 0.f);
  }
}

template <class T, int S, int NT, int MT, bool XL, int MODE>
hipError_t rows_launch_one(const I8Args& a, const I8Group& g, int64_t mtiles, const RowsPlan& l, int mshift, hipStream_t s) {
  const auto kern = &i8_rows_kernel<T, S, NT, MT, XL, MODE>;
  if (l.bytes > 60 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, kRowsLds);
    if (e != hipSuccess) return e;
  }
  const int tiles = (a.N + 15) / 16, per = NT / S * l.cg;
  hipLaunchKernelGGL(kern, dim3((unsigned)((tiles + per - 1) / per), (unsigned)mtiles), dim3(l.kw * l.cg * kWave),
                     l.bytes, s, a, g, __builtin_ctz(l.kw), mshift, l.xstride);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Many rows: tiles of BM rows by BN columns (of two weights BN / 2 of each),
// chunks of 128 k through a ring of R in LDS.  The weight is the MFMA's first
// operand, so that a lane's four sums are of one row; which columns a tile's 16
// operand rows are is chosen so that a lane's sums of its NT tiles are 4 NT
// neighbouring columns.  Scaled sums leave through the ring's LDS, so that a
// lane's results are pieces of 16 bytes.  A chunk's copies are issued R - 1 chunks
// ahead, its operands read from LDS a step of 64 k before they are multiplied.
// 4,096^3 with x in 8 bits 67 us (2.04 POPS) where a library's product without
// scales takes 75: the matrix cores are busy 53% of the CUs' cycles, LDS has no
// conflicts, waves wait 30% of theirs.  Tiles of 64 x 64 are bound by what L2 gives
// a CU, about 80 bytes/ns or 0.2 us a chunk (203 x 4,080 -> 4,093: 11.5 us).
// Where tiles are few, several workgroups share one, each with a
// part of k, leave their sums in a workspace, and a second kernel adds them.
// ---------------------------------------------------------------------------
template <class T, int S, int BM, int BN, int WM, int WN, int R, int EU, int MODE>
__global__ __launch_bounds__(64 * WM * WN, EU) void i8_tile_kernel(I8Args p, I8Group g, int mtiles, int ntiles) {
  constexpr int NW = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16, NS = NT / S;
  constexpr int XI = BM / 8 / NW, WI = BN / 8 / NW, NI = XI + WI;  // copies of 1 KiB a wave and chunk
  constexpr int XB = BM * kChunk, SLOT = XB + BN * kChunk;
  constexpr int SB = BN / 16 / S;  // blocks of a weight in a chunk's half
  static_assert(NW % 2 == 0 && XI * 8 * NW == BM && WI * 8 * NW == BN && WI % 2 == 0, "copies");
  static_assert(BM <= 64 * NW && BN <= 64 * NW, "a thread for each row and column");
  // One array for all: with several the compiler waits for every copy in flight before it reads the ring
  // (64 x 64: 0.6 us a chunk instead of 0.29).
  __shared__ __attribute__((aligned(1024))) char mem[R * SLOT + BN * 8 + BM * (MODE == DOWN ? 8 : 4)];
  GP_LDS char* const lds = (GP_LDS char*)mem;
  GP_LDS float* const colscale = (GP_LDS float*)(lds + R * SLOT);  // of the tile's columns, a weight's after the other's
  GP_LDS float* const colbias = colscale + BN;
  GP_LDS float* const rowscale = colbias + BN;
  GP_LDS int* const rowpair = (GP_LDS int*)(rowscale + BM);
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;
  const int N = p.N, K = p.K, K64 = (K + 63) / 64, N16 = (N + 15) / 16, chunks = (K + kChunk - 1) / kChunk;
  const int kb = wave & 1;  // of a chunk's two blocks along k
  // Experts' tiles are counted by the plan, whose tiles this one may be a part of.
  if constexpr (MODE != DENSE) mtiles = g.info[0] << g.shift;
  const int total = mtiles * ntiles;
  if ((int)blockIdx.x >= total) return;

  // A workgroup of 256 x 256 has its CU for itself, and takes one tile after the
  // other, every gridDim.x-th; where two share a CU, one's beginnings and ends
  // lie under the other's chunks, and a workgroup for every tile is better
  // (8,192^3 with tiles of 64: 839 us, one after the other 907).
  constexpr bool LOOP = BM == 256;
  int64_t m0;
  int rows, nb0;  // rows there are; first block of columns
  __amdgpu_buffer_rsrc_t xr, wr0, wr1;
  unsigned xo[XI], wo[WI];
  // of row and column tid
  float rs, cs, cb;
  int rp;
  auto setup = [&](int b) {
    const int lane = opaque(threadIdx.x & 63), tid = opaque(threadIdx.x);  // offsets are made anew: there are no registers to keep them
    // Neighbours of one XCD take eight row tiles of a column tile, then of the next.
    const int id = xcd_order(b, total);
    const int gm0 = id / (8 * ntiles) * 8, rest = id % (8 * ntiles);
    const int gm = mtiles - gm0 < 8 ? mtiles - gm0 : 8, mt = gm0 + rest % gm;
    nb0 = rest / gm * SB;
    int64_t expert = 0;
    if constexpr (MODE == DENSE) {
      m0 = (int64_t)mt * BM;
      rows = p.M - m0 < BM ? (int)(p.M - m0) : BM;
    } else {
      const TileRec rec = g.tiles[mt >> g.shift];
      const int part = (mt & ((1 << g.shift) - 1)) * BM;
      m0 = rec.row0 + part;
      rows = rec.rows - part < BM ? rec.rows - part : BM;  // 0 and less: a part behind the rows
      rows = rows < 0 ? 0 : rows;
      expert = rec.expert;
    }
    xr = MODE == UP ? make_rsrc(p.xq, (int)(p.M * K)) : make_rsrc((const char*)p.xq + m0 * K, rows * K);
    wr0 = make_rsrc((const char*)p.side[0].wq + expert * g.wbytes, N16 * K64 * 1024);
    wr1 = make_rsrc((const char*)p.side[S - 1].wq + expert * g.wbytes, N16 * K64 * 1024);
    // Copies.  x: eight rows each, piece c of row r at c ^ (r / 2) % 8.  Weight:
    // one block each, piece q of local block l at q ^ 4 (l % 4), which keeps the
    // sixteen columns that an operand takes from several blocks in different banks.
    int tok[XI];
    if constexpr (MODE == UP) {  // loads under a condition each would be waited for one by one
      const auto tr = make_rsrc(g.tok + m0, rows * 4);
#pragma unroll
      for (int q = 0; q < XI; ++q)
        tok[q] = (int)__builtin_amdgcn_raw_buffer_load_b32(tr, (8 * (q * NW + wave) + (lane >> 3)) * 4, 0, 0);
    }
#pragma unroll
    for (int q = 0; q < XI; ++q) {
      const int row = 8 * (q * NW + wave) + (lane >> 3);
      const unsigned piece = (unsigned)(((lane & 7) ^ ((row >> 1) & 7)) << 4);
      xo[q] = (unsigned)(MODE == UP ? tok[q] : row) * (unsigned)K + piece;
      if (MODE == UP && row >= rows) xo[q] = 0x80000000u;
    }
#pragma unroll
    for (int q = 0; q < WI; ++q) {
      const int l = (q * NW + wave) >> 1, n16 = nb0 + l % SB;
      wo[q] = n16 < N16 ? (unsigned)(n16 * K64 + kb) * 1024u + (unsigned)((lane ^ (4 * (l & 3))) << 4) : 0xC0000000u;
    }
    // What the epilogue needs of each row and column, a thread each; it goes to LDS when the last tile's is done with.
    rs = cs = cb = 0.f, rp = 0;
    if (tid < rows) {
      rs = p.xs[MODE == UP ? g.tok[m0 + tid] : m0 + tid];
      if (MODE == DOWN) rp = g.pair[m0 + tid];
    }
    const int s = tid / (BN / S), n = nb0 * 16 + tid % (BN / S);
    if (tid < BN && n < N) {
      const I8Side d = s ? p.side[S - 1] : p.side[0];
      cs = d.s[expert * N + n];
      if (MODE == DENSE && d.b) cb = T::val(((const half_t*)d.b)[n]);
    }
  };
  auto publish = [&] {
    if (tid < BM) {
      rowscale[tid] = rs;
      if (MODE == DOWN) rowpair[tid] = rp;
    }
    if (tid < BN) colscale[tid] = cs, colbias[tid] = cb;
  };
  auto issue = [&](int c, int c1, int slot) {
    GP_LDS char* at = lds + slot * SLOT;
    const bool in = c < c1;
#pragma unroll
    for (int q = 0; q < XI; ++q)
      dma16_buf(xr, (int)(in ? xo[q] + (unsigned)c * kChunk : kNowhere), at + (q * NW + wave) * 1024);
    const bool win = in && 2 * c + kb < K64;
#pragma unroll
    for (int q = 0; q < WI; ++q)
      dma16_buf(S == 2 && q >= WI / 2 ? wr1 : wr0, (int)(win ? wo[q] + (unsigned)c * 2048u : kNowhere),
                at + XB + (q * NW + wave) * 1024);
  };
  // Operands.
  int xa[2], wa[S][NS];
#pragma unroll
  for (int h = 0; h < 2; ++h) xa[h] = (wm * MT * 16 + j) * 128 + (((4 * h + lg) ^ ((j >> 1) & 7)) << 4);
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      const int n = 4 * NS * (j >> 2) + 4 * t + (j & 3), l = s * SB + wn * NS + (n >> 4);
      wa[s][t] = XB + l * 2048 + (((lg * 16 + (n & 15)) ^ (4 * (l & 3))) << 4);
    }

  const int per = (chunks + gridDim.y - 1) / gridDim.y, c0 = blockIdx.y * per;
  const int c1 = c0 + per < chunks ? c0 + per : chunks;
  // A chunk is multiplied in steps: half of its k, and with eight row tiles half
  // of them.  A step's operands are read from LDS while the step before it is
  // multiplied, a chunk's first ones too: at its last step every operand of the
  // chunk is in registers, so that behind one barrier its slot takes the chunk R
  // further on and the next slot is read.
  constexpr int G = MT > 4 ? 2 : 1, MG = MT / G, STEPS = 2 * G;

  int b = blockIdx.x;
  setup(b);
  if (!LOOP && MODE != DENSE && rows <= 0) return;  // a plan's tile may end before its last part
#pragma unroll
  for (int i = 0; i < R; ++i) issue(c0 + i, c1, i);
  publish();
#pragma unroll 1
  for (;;) {
    i32x4 acc[S][NS][MT] = {};
    u32x4 w[2][S][NS], x[2][MG];
    auto read = [&](int q, GP_LDS const char* slot) {  // step q of the chunk in slot
      const int h = q / G;
      if (q % G == 0) {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int t = 0; t < NS; ++t) w[h][s][t] = *(GP_LDS const u32x4*)(slot + wa[s][t] + h * 1024);
      }
#pragma unroll
      for (int m = 0; m < MG; ++m) x[q & 1][m] = *(GP_LDS const u32x4*)(slot + xa[h] + (q % G * MG + m) * 2048);
    };
    wait_vmcnt<(R - 1) * NI>();
    lds_barrier();
    read(0, lds);
    int at = 0, c = c0;
    // A wave behind the last row only copies.  (In the smaller kernels this branch makes the compiler wait for a step's
    // reads at once: 128 rows of 4,096 from 4,096 11.0 us instead of 10.3.)
    if (LOOP && wm * MT * 16 >= rows) {
#pragma unroll 1
      for (; c < c1; ++c) {
        wait_vmcnt<(R - 2) * NI>();
        lds_barrier();
        issue(c + R, c1, at);
        at = at + 1 == R ? 0 : at + 1;
      }
    }
#pragma unroll 1
    for (; c < c1; ++c) {
      GP_LDS const char* slot = lds + at * SLOT;
#pragma unroll
      for (int q = 0; q < STEPS; ++q) {
        if (q + 1 < STEPS) {
          read(q + 1, slot);
        } else {
          wait_vmcnt<(R - 2) * NI>();
          lds_barrier();
          issue(c + R, c1, at);
          at = at + 1 == R ? 0 : at + 1;
          read(0, lds + at * SLOT);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int m = 0; m < MG; ++m)
#pragma unroll
          for (int s = 0; s < S; ++s)
#pragma unroll
            for (int t = 0; t < NS; ++t)
              acc[s][t][q % G * MG + m] = mma8(w[q / G][s][t], x[q & 1][m], acc[s][t][q % G * MG + m]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    wait_vmcnt<0>();
    lds_barrier();  // every wave is done with the ring

    if (MODE == DENSE && gridDim.y > 1) {
      // a lane's columns: 4 NS from n0 of each weight, of row j of each row tile
      const int n0 = nb0 * 16 + wn * (16 * NS) + 4 * NS * lg;
      int* const part = (int*)p.part + (int64_t)blockIdx.y * S * p.M * N;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int row = wm * MT * 16 + m * 16 + j;
        if (row >= rows) continue;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          int* to = part + ((int64_t)s * p.M + m0 + row) * N + n0;
#pragma unroll
          for (int t = 0; t < NS; ++t) {
            if (n0 + 4 * t + 4 <= N)
              *(i4u*)(to + 4 * t) = acc[s][t][m];
            else
#pragma unroll
              for (int e = 0; e < 3; ++e)
                if (n0 + 4 * t + e < N) to[4 * t + e] = acc[s][t][m][e];
          }
        }
      }
      return;  // such a launch has a workgroup for every tile
    }

    // The next tile's first chunk, where there is one, is copied while this one leaves through the
    // other slots: a wave's sums through its own part of them, eight neighbouring
    // columns of a row a lane then, whole lines a wave, and a short rolled loop with
    // the epilogue once (code is fetched from memory: with the epilogue unrolled over
    // a lane's sums, and loads under conditions, a tile of 256 x 256 took 18 us
    // besides its chunks).  Piece c of four sums of row r lies at c ^ r.
    constexpr int OC = 16 * NS, NP = 4 * NS * S;  // a wave's columns of out; pieces a row
    constexpr int ROOM = (R - 1) * SLOT / (NW * 16 * NP * 16), HM = ROOM >= MT ? MT : ROOM >= 4 ? 4 : ROOM >= 2 ? 2 : 1;
    static_assert(ROOM >= 1, "a row tile's sums fit the other slots");
    constexpr int LPR = OC / 8, RPI = 64 / LPR;  // lanes a row, rows a turn
    const int lane = opaque(threadIdx.x & 63), j = lane & 15, lg = lane >> 4;
    const int64_t out0 = m0;
    const int last = rows, oc = lane % LPR, orow = lane / LPR, col = wn * OC + oc * 8;
    const int n = nb0 * 16 + col, cnt = N - n < 8 ? N - n : 8;
    b += gridDim.x;
    const bool more = LOOP && b < total;
    if (more) {
      setup(b);
      issue(c0, c1, 0);
    }
    GP_LDS char* const mine = lds + SLOT + wave * (HM * 16 * NP * 16);
    float sc[S][8], bias[S][8] = {};
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f4 v = *(GP_LDS const f4*)(colscale + s * (BN / S) + col + 4 * h);
        f4 b = {};
        if constexpr (MODE == DENSE) b = *(GP_LDS const f4*)(colbias + s * (BN / S) + col + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[s][4 * h + e] = v[e], bias[s][4 * h + e] = b[e];
      }
#pragma unroll
    for (int part = 0; part < MT / HM; ++part) {
#pragma unroll
      for (int m = 0; m < HM; ++m)
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int t = 0; t < NS; ++t)
            *(GP_LDS i32x4*)(mine + (m * 16 + j) * (NP * 16) + (((s * 4 * NS + NS * lg + t) ^ (j & (NP - 1))) << 4)) =
                acc[s][t][part * HM + m];
      const int row0 = wm * MT * 16 + part * HM * 16;
#pragma unroll 1
      for (int it = 0; it < HM * 16; it += RPI) {
        const int lrow = it + orow, row = row0 + lrow;
        if (row >= last || cnt <= 0) continue;
        const float xsc = rowscale[row];
        float v[8], u[8];
        auto take = [&](int s, float (&to)[8]) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const i32x4 a = *(GP_LDS const i32x4*)(mine + lrow * (NP * 16) +
                                                   (((s * 4 * NS + 2 * oc + h) ^ (lrow & (NP - 1))) << 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) to[4 * h + e] = (float)a[e] * sc[s][4 * h + e] * xsc;
          }
        };
        take(0, v);
        if constexpr (MODE == DOWN) {  // N a multiple of 16 here
          float* const to = (float*)p.out + (int64_t)rowpair[row] * N + n;
          *(f4*)to = f4{v[0], v[1], v[2], v[3]};
          *(f4*)(to + 4) = f4{v[4], v[5], v[6], v[7]};
        } else {
          if constexpr (S == 2) take(1, u);
          finish8<T, S, MODE == DENSE>(p, out0 + row, n, cnt, v, u, bias);
        }
      }
    }
    if (!more) return;
    lds_barrier();  // the other slots, and the rows' and columns' values, are done with
#pragma unroll
    for (int i = 1; i < R; ++i) issue(c0 + i, c1, i);
    publish();
  }
}

// The parts of k added, and the epilogue: eight columns of a row a thread.
template <class T, int S>
__global__ __launch_bounds__(256) void i8_join_kernel(I8Args p, int parts) {
  const int pieces = (p.N + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.M * pieces) return;
  const int64_t m = i / pieces;
  const int n = (int)(i - m * pieces) * 8, cnt = p.N - n < 8 ? p.N - n : 8;
  int a[S][8] = {};
#pragma unroll 4
  for (int k = 0; k < parts; ++k)
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int* at = (const int*)p.part + (((int64_t)k * S + s) * p.M + m) * p.N + n;
      if (cnt >= 8) {
        const i4u lo = *(const i4u*)at, hi = *(const i4u*)(at + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[s][e] += lo[e], a[s][4 + e] += hi[e];
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (e < cnt) a[s][e] += at[e];
      }
    }
  const float xsc = p.xs[m];
  float v[8], u[8], sc[S][8], b[S][8] = {};
#pragma unroll
  for (int s = 0; s < S; ++s) {
    load_scales8(p.side[s].s, n, p.N, sc[s]);
    if (p.side[s].b) load_row8<T>((const half_t*)p.side[s].b, n, cnt, p.N, b[s]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = (float)a[0][e] * sc[0][e] * xsc;
    u[e] = (float)a[S - 1][e] * sc[S - 1][e] * xsc;
  }
  finish8<T, S>(p, m, n, cnt, v, u, b);
}

// ---------------------------------------------------------------------------
// Which kernel
// ---------------------------------------------------------------------------
struct TilePlan {
  int size, parts;  // 64, 128 or 256; parts of k
};

// The time of a product of `tiles` tiles on tiles, in us: a chunk takes one
// workgroup of a CU `alone`, and the two that share a CU `pair` (256 x 256: has
// a CU by itself, and takes longer where it fills the chip, whose power is then the limit),
// and what is not chunks takes `fixed` a turn.  Measured, K 4,096 (M x N: 64,
// 128, 256):  512 x 4,096 16.4, 24.5, 52;  1,024 x 4,096 29.8, 27.1, 52.7;
// 4,096 x 4,096 108, 75, 64;  the estimate: 16.5, 25.5, 49.6;  29.6, 25.5, 49.6;  107, 75, 64.
float tile_time(int size, int64_t tiles, int chunks, int num_cus) {
  const int64_t n = (tiles + num_cus - 1) / num_cus;  // workgroups of the fullest CU
  if (size == 256) return (float)n * (8.f + (float)chunks * (tiles * 2 > num_cus ? 1.74f : 1.3f));
  const float alone = size == 128 ? 0.64f : 0.2f, pair = size == 128 ? 1.05f : 0.4f;
  return 4.f + (float)(n / 2 + n % 2) + (float)chunks * ((float)(n / 2) * pair + (float)(n % 2) * alone);
}

TilePlan tile_plan(int64_t M, int N, int K, int sides, int num_cus) {
  const int chunks = (K + kChunk - 1) / kChunk;
  TilePlan best{256, 1};
  float least = 0.f;
  for (int size : {256, 128, 64}) {
    const int64_t cols = size / sides, tiles = (M + size - 1) / size * ((N + cols - 1) / cols);
    for (int parts = 1; parts <= 16 && parts <= chunks; ++parts) {
      float t = tile_time(size, tiles * parts, (chunks + parts - 1) / parts, num_cus);
      // the second kernel, and the sums' way to memory and back
      if (parts > 1) t += 3.f + (float)parts * (float)M * (float)N * (float)sides * 8.f / 4e6f;
      if (least == 0.f || t < least) best = TilePlan{size, parts}, least = t;
    }
  }
  return best;
}

// Products that run on tiles: up to 64 rows those whose x the kernel for few rows
// would read for too many columns.  In us, on tiles / by the kernel for few rows:
//   32 rows: 4,096 columns from 4,096 k 10.8 / 6.5, from 16,384 17.1 / 13.4, 16,384 from 4,096 13.0 / 16.3,
//            2 x 16,384 28.7 / 36.7
//   48 and 64 rows: 4,096 from 4,096 9.7 / 9.2, 8,192 from 8,192 16.9 / 18.4, 16,384 from 4,096 13.2 / 19.3,
//            2 x 8,192 from 2,048 12.4 / 15.6, 2 x 16,384 from 4,096 29.6 / 43.0
//   16 rows: 8,192 from 8,192 18.5 / 15.2, 16,384 from 4,096 12.7 / 12.9
bool on_tiles(int64_t M, int N, int sides) {
  const int64_t n = (int64_t)N * sides;
  return M > 64 || (M > 32 && n > 4096) || (M > 16 && n > 8192);
}

// Tokens whose experts run by themselves: two, or up to eight where most of them
// will have different ones (an expert that two tokens choose is read twice, but the
// plan, h's bytes and the sums are no launches of their own).  In us, so / with a plan:
//   8 of 64 experts of 2,048 x 1,024:  2 tokens 28 / -, 4 43.3 / 52.6, 6 60.3 / 65.6, 8 73.8 / 72.2
//   4 of 16 of 2,048 x 4,096:  3 58.4 / 57.8, 4 69.9 / 68.9, 8 124.7 / 78.7;  2 of 32 of 1,024 x 512:  8 14.0 / 22.2
bool few_tokens(int64_t T, int E, int topk) { return T <= 2 || (T <= 8 && 4 * T * topk <= 3 * E); }

// Rows of 16-bit x that the kernel for few rows makes bytes of itself: up to four (three as four) of 16,384 values together.
bool own_bytes(int64_t M, int K) { return M <= 4 && K * (M <= 1 ? 1 : M <= 2 ? 2 : 4) <= 16384; }

// mtiles: of 16 mt rows.  A product of experts (MODE) has them from its plan; busy: those that are worth counting.
template <class T, int S, int MODE>
hipError_t rows_launch(const I8Args& a, const I8Group& g, int mt, int64_t mtiles, int64_t busy, bool x16, int num_cus,
                       hipStream_t s) {
  RowsPlan l{};
  l.xl = x16;
  l.mt = mt;
  const int chunks = (a.K + kChunk - 1) / kChunk, rows = MODE == DENSE ? (int)a.M : 1;
  const int64_t tiles = (int64_t)((a.N + 15) / 16) * S * busy;
  // Tiles a workgroup: as many as leave every CU a workgroup, so that x is read for
  // more columns at once; of one row, whose bytes cost little, every CU two, of
  // eight waves, one's bytes and sums under the other's copies (one row / four rows with two and with one: 16,384
  // columns from 4,096 k 12.4 / 14.7 and 12.8 / 13.4 us, 8,192 from 8,192 12.2 and 13.0).
  const int64_t full = (int64_t)num_cus * (l.xl && rows == 1 ? 2 : 1);
  int per = l.mt == 1 && tiles >= 4 * full ? 4 : tiles >= 2 * full ? 2 : 1;
  if (per < S) per = S;
  l.nt = per > 2 ? 2 : per;
  const int waves = rows_waves(l.nt, l.mt, l.xl);
  const int ring = rows_ring(l.nt, l.mt, l.xl) * slot_bytes(l.nt, l.mt, l.xl);
  const int mshift = rows <= 1 ? 0 : rows <= 2 ? 1 : 2;
  l.xstride = (chunks * kChunk + 255) / 256 * 256 + 64;
  int xbytes = 0;
  if (l.xl) {
    // the workgroup's threads make the bytes: as many waves as there can be, but no more than chunks and x need
    int need = 1;
    while (need * kWave * 32 < (a.K << mshift) || need < (1 << mshift)) need *= 2;
    xbytes = l.xstride << mshift;
    l.cg = per / l.nt;
    l.kw = waves / l.cg;
    const bool two = tiles / per >= 2 * num_cus;
    while (l.kw > 1 && (l.kw / 2 >= chunks || (two && l.kw * l.cg > 8)) && l.kw / 2 * l.cg >= need) l.kw /= 2;
  } else {
    // k over as many waves as fill the chip with eight a CU; workgroups of four waves and more
    l.kw = waves;
    while (l.kw > 1 && (l.kw / 2 >= chunks || tiles / l.nt * (l.kw / 2) >= 8 * num_cus)) l.kw /= 2;
    l.cg = l.kw < 4 ? 4 / l.kw : 1;
  }
  l.bytes = l.kw * l.cg * ring + xbytes;
#define GP_CASE(n, m)                                                                         \
  if constexpr (n >= S && (m == 1 || MODE == DENSE))                                          \
    if (l.nt == n && l.mt == m) {                                                             \
      if constexpr (m == 1 && MODE != DOWN)                                                   \
        if (l.xl) return rows_launch_one<T, S, n, m, true, MODE>(a, g, mtiles, l, mshift, s); \
      return rows_launch_one<T, S, n, m, false, MODE>(a, g, mtiles, l, mshift, s);            \
    }
  GP_CASE(1, 1) GP_CASE(2, 1) GP_CASE(1, 2) GP_CASE(2, 2) GP_CASE(1, 4) GP_CASE(2, 4)
#undef GP_CASE
  return hipErrorInvalidValue;
}

template <class T, int S, int MODE>
hipError_t tile_launch(const I8Args& a, const I8Group& g, int64_t mtiles, const TilePlan& plan, int num_cus, hipStream_t s) {
  const int64_t cols = plan.size / S, ntiles = (a.N + cols - 1) / cols, fit = plan.size == 256 ? num_cus : int64_t(1) << 31;
  if (mtiles * ntiles >= int64_t(1) << 31) return hipErrorInvalidValue;
  // of 256 x 256 as many workgroups as the chip holds; one for every tile else, and where k is in parts
  const int64_t wgs = plan.parts > 1 || mtiles * ntiles < fit ? mtiles * ntiles : fit;
  if (wgs * (plan.size == 256 ? 512 : 256) >= int64_t(1) << 32) return hipErrorInvalidValue;  // more threads than a launch holds
  const dim3 grid((unsigned)wgs, (unsigned)plan.parts);
#define GP_TILE(size, wm, wn, r)                                                                                  \
  hipLaunchKernelGGL((i8_tile_kernel<T, S, size, size, wm, wn, r, 2, MODE>), grid, dim3(64 * wm * wn), 0, s, a, g, \
                     (int)mtiles, (int)ntiles)
  if (plan.size == 256) GP_TILE(256, 2, 4, 2);
  else if (plan.size == 128) GP_TILE(128, 2, 2, 2);
  else GP_TILE(64, 2, 2, 4);
#undef GP_TILE
  const hipError_t e = hipGetLastError();
  if constexpr (MODE == DENSE) {
    if (e != hipSuccess || plan.parts == 1) return e;
    const int64_t pieces = a.M * ((a.N + 7) / 8);
    hipLaunchKernelGGL((i8_join_kernel<T, S>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, a, plan.parts);
    return hipGetLastError();
  }
  return e;
}

// The workspace: bytes and scales of 16-bit rows, then the parts' sums.
struct Layout {
  int64_t xs, part, bytes;
};
Layout layout(int64_t M, int N, int K, bool x16, int sides, int num_cus) {
  Layout l{};
  if (x16 && !own_bytes(M, K)) {
    l.xs = (M * K + 255) / 256 * 256;
    l.part = (l.xs + M * 4 + 255) / 256 * 256;
  }
  l.bytes = l.part;
  if (on_tiles(M, N, sides)) {
    const TilePlan p = tile_plan(M, N, K, sides, num_cus);
    if (p.parts > 1) l.bytes += (int64_t)p.parts * sides * M * N * 4;
  }
  return l;
}

template <class T, int S>
hipError_t launch(I8Args a, int num_cus, hipStream_t s) {
  const bool x16 = !a.xs, xl = x16 && own_bytes(a.M, a.K);
  const Layout l = layout(a.M, a.N, a.K, x16, S, num_cus);
  if (x16 && !xl) {
    a.xq = (char*)a.ws;
    a.xs = (float*)((char*)a.ws + l.xs);
    const hipError_t e = rows_to_bytes_launch<T>(a.x, a.M, a.K, (char*)a.ws, (float*)a.xs, s);
    if (e != hipSuccess) return e;
  }
  if (!on_tiles(a.M, a.N, S)) {
    const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
    const int64_t mtiles = (a.M + 16 * mt - 1) / (16 * mt);
    return rows_launch<T, S, DENSE>(a, I8Group{}, mt, mtiles, mtiles, xl, num_cus, s);
  }
  a.part = (char*)a.ws + l.part;
  const TilePlan plan = tile_plan(a.M, a.N, a.K, S, num_cus);
  return tile_launch<T, S, DENSE>(a, I8Group{}, (a.M + plan.size - 1) / plan.size, plan, num_cus, s);
}

// ---------------------------------------------------------------------------
// A feed-forward block of experts.  out[t] = r[t] + sum over j of w[t][j] *
// Down(act(x Wg) * (x Wu)) of expert ids[t][j].
//
// The pairs (token, choice) are put in order of their experts, so that an
// expert's rows are one product; its rows are tokens of x, which the first
// product gathers while it copies them.  The pairs' results go back to their
// places in fp32 and are added in the order of the choices: nothing depends on
// the order in which workgroups end.
// ---------------------------------------------------------------------------

// One workgroup an expert: counts of all experts (whole numbers, in LDS), where
// the expert's rows and tiles begin, and its pairs in their order.  Whole tiles
// come first and the experts' last, shorter ones behind all of them.  Loads of
// ids are in batches, and up to 8,192 pairs stay in registers for the second
// pass: one after the other they were 12 us for 8,192 pairs of 8 experts.
// The workgroups behind the experts' make the tokens' rows bytes meanwhile.
template <class T, int WPR>
__global__ __launch_bounds__(1024) void i8_plan_kernel(const int* ids, int64_t P, int E, int topk, int tile, TileRec* tiles,
                                                      int* info, int* tok, int* pair, const half_t* x, int H, char* q,
                                                      float* xs) {
  constexpr int B = 8, SUMS = 6;
  if ((int)blockIdx.x >= E) {
    __shared__ unsigned part[16];
    rows_to_bytes<T, 4, WPR, 16>(x, P / topk, H, q, xs, nullptr, blockIdx.x - E, part);
    return;
  }
  __shared__ int count[kExpertsMaxE];
  __shared__ int own[16], sums[16][SUMS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e = blockIdx.x;
  if (tid < E) count[tid] = 0;
  __syncthreads();
  const int64_t seg = ((P + 15) / 16 + 63) / 64 * 64, lo = wave * seg, hi = lo + seg < P ? lo + seg : P;
  const auto r = make_rsrc(ids, (int)(P * 4));
  int id[B];
  auto load = [&](int64_t base) {
#pragma unroll
    for (int q = 0; q < B; ++q) id[q] = (int)__builtin_amdgcn_raw_buffer_load_b32(r, (int)((base + q * 64 + lane) * 4), 0, 0);
#pragma unroll
    for (int q = 0; q < B; ++q) id[q] = base + q * 64 + lane < hi ? id[q] : -1;
  };
  int mine = 0;
  for (int64_t base = lo; base < hi; base += B * 64) {
    load(base);
#pragma unroll
    for (int q = 0; q < B; ++q) {
      if ((unsigned)id[q] < (unsigned)E) atomicAdd(&count[id[q]], 1);
      mine += __popcll(__ballot(id[q] == e));
    }
  }
  if (lane == 0) own[wave] = mine;
  __syncthreads();
  // of the experts before this one, and of all: rows, whole tiles, shorter ones
  const int c = tid < E ? count[tid] : 0, n = c / tile, m = c % tile ? 1 : 0;
  const bool before = tid < e;
  int v[SUMS] = {before ? c : 0, before ? n : 0, before ? m : 0, c, n, m};
#pragma unroll
  for (int k = 0; k < SUMS; ++k) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v[k] += __shfl_xor(v[k], d);
    if (lane == 0) sums[wave][k] = v[k];
  }
  __syncthreads();
  int t[SUMS] = {}, at = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
#pragma unroll
    for (int k = 0; k < SUMS; ++k) t[k] += sums[w][k];
    at += w < wave ? own[w] : 0;
  }
  const int row0 = t[0], rows = count[e], whole = rows / tile;
  if (e == 0 && tid == 0) info[0] = t[4] + t[5], info[1] = t[3];
  for (int i = tid; i < whole; i += 1024) tiles[t[1] + i] = TileRec{e, row0 + i * tile, tile, 0};
  if (tid == 0 && rows % tile) tiles[t[4] + t[2]] = TileRec{e, row0 + whole * tile, rows % tile, 0};
  if (mine == 0) return;
  at += row0;
  for (int64_t base = lo; base < hi; base += B * 64) {
    if (seg > B * 64) load(base);
#pragma unroll
    for (int q = 0; q < B; ++q) {
      const unsigned long long b = __ballot(id[q] == e);
      if (id[q] == e) {
        const int to = at + __popcll(b & ((1ull << lane) - 1)), p = (int)(base + q * 64 + lane);
        tok[to] = p / topk;
        pair[to] = p;
      }
      at += __popcll(b);
    }
  }
}

// The pairs' results times their weights, in the order of the choices, and r:
// eight columns of a token a thread.  Bound by the results' loads: 4,096 tokens
// of two choices and 2,048 columns 17.5 us (with r 101 MB, 5.8 TB/s).
template <class T>
__global__ __launch_bounds__(256) void i8_combine_kernel(ExpertsArgs p, const float* y) {
  const int pieces = p.H / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.T * pieces) return;
  const int64_t t = i / pieces;
  const int n = (int)(i - t * pieces) * 8;
  float v[8] = {}, f[8];
#pragma unroll 4
  for (int j = 0; j < p.topk; ++j) {
    const int64_t at = t * p.topk + j;
    if ((unsigned)p.ids[at] >= (unsigned)p.E) continue;
    const float w = p.weights[at];
    const f4 lo = *(const f4*)(y + at * p.H + n), hi = *(const f4*)(y + at * p.H + n + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(w, lo[e], v[e]), v[4 + e] = __builtin_fmaf(w, hi[e], v[4 + e]);
  }
  if (p.r) {
    load8<T>((const half_t*)p.r + t * p.H + n, 8, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += f[e];
  }
  store8<T>((half_t*)p.out + t * p.H + n, 8, v);
}

// A few tokens' second half and their sums in one launch: wave (choice, kw) of a
// token's workgroup multiplies its share of k of its choice's expert with the
// workgroup's COLS columns, and the choices are added in their order.  With
// eight columns a workgroup takes half of each block, whole lines still, so that
// twice as many CUs have work.  A token's 4 of 16 experts of 4,096 x 2,048 9.3 us
// (34 MB, 3.6 TB/s; 6.8 at a large copy's rate), the rows' bytes before the products
// and the sums behind them among it.
constexpr int kTokenRing = 2;
constexpr int kTokenSlot = 2048;  // bytes of a wave's ring: 128 k of sixteen columns or 256 of eight
constexpr int kTokenPieces = 8;   // of eight values a thread makes bytes of

template <class T, int COLS>
__global__ __launch_bounds__(1024) void i8_token_down_kernel(ExpertsArgs p, const half_t* h, int64_t wbytes, int kwshift,
                                                            int xstride) {
  constexpr int KB = 32 / COLS, XP = kTokenPieces;  // blocks of 64 k a slot
  __shared__ unsigned tops[16];
  __shared__ float hs[16];
  __shared__ int part[16][COLS];
  GP_LDS char* lds = dyn_lds();
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, lg = lane >> 4;
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KW = 1 << kwshift, kw = wave & (KW - 1), slot = wave >> kwshift;
  const int F = p.F, K64 = (F + 63) / 64, steps = (K64 + KB - 1) / KB;
  const int64_t t = blockIdx.y, pair = t * p.topk + slot;
  const int n0 = xcd_order(blockIdx.x, gridDim.x) * COLS, n16 = n0 >> 4;
  const int e = p.ids[pair];
  const bool valid = (unsigned)e < (unsigned)p.E;

  const int tpr = KW * 64, at = (tid - slot * tpr) * 8;
  u32x4 v[XP];
  const auto hr = make_rsrc(h + pair * F, valid ? F * 2 : 0);  // what lies there for an id of no expert is not read
#pragma unroll
  for (int i = 0; i < XP; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(hr, (at + i * tpr * 8) * 2, 0, 0);
  const auto wr = make_rsrc((const char*)p.wd + (valid ? e : 0) * wbytes, valid ? (int)wbytes : 0);
  GP_LDS char* const ring = lds + wave * (kTokenRing * kTokenSlot);
  // a copy: lane l fetches column l % COLS of block l / (4 COLS)
  const int lb = lane / (4 * COLS), lp = lane % (4 * COLS);
  const unsigned wo = (unsigned)(n16 * K64 + lb) * 1024u + (unsigned)((lp / COLS * 16 + (n0 & 15) + lp % COLS) * 16);
  auto issue = [&](int c, int at) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int b = c * KB + i * (KB / 2);
      dma16_buf(wr, (int)(b + lb < K64 ? wo + (unsigned)b * 1024u : kNowhere), ring + at * kTokenSlot + i * 1024);
    }
  };
#pragma unroll
  for (int i = 0; i < kTokenRing; ++i) issue(kw + i * KW, i);

  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < XP; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) top = top2(top, v[i][k]);
  top = wave_top(top);
  if (lane == 0) tops[wave] = top;
  lds_barrier();
  top = wave_top(tops[(slot << kwshift) + (lane & (KW - 1))]);
  const RowScale sc = row_scale<T>(top);
  GP_LDS char* const xl = lds + waves * (kTokenRing * kTokenSlot) + slot * xstride;
#pragma unroll
  for (int i = 0; i < XP; ++i) {
    const int k = at + i * tpr * 8;
    if (k < F) *(GP_LDS u32x2*)(xl + k) = round8<T>(v[i], sc);
  }
  if (at == 0) hs[slot] = sc.scale;
  lds_barrier();

  i32x4 acc = {};
  int s = 0;
  for (int c = kw; c < steps; c += KW) {
    wait_vmcnt<(kTokenRing - 1) * 2>();
    compiler_fence();
    u32x4 a[KB], b[KB];
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      a[i] = *(GP_LDS const u32x4*)(xl + (c * KB + i) * 64 + lg * 16);
      b[i] = *(GP_LDS const u32x4*)(ring + s * kTokenSlot + (i * 4 * COLS + lg * COLS + (j & (COLS - 1))) * 16);
    }
    compiler_fence();
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    issue(c + kTokenRing * KW, s);
    s = s + 1 == kTokenRing ? 0 : s + 1;
#pragma unroll
    for (int i = 0; i < KB; ++i) acc = mma8(a[i], b[i], acc);
  }
  wait_vmcnt<0>();
  if (lane < COLS) part[wave][lane] = acc[0];  // every row of the operand was the same
  __syncthreads();
  const int n = n0 + tid;
  if (tid < COLS && n < p.H) {
    float out = 0.f;
    for (int k = 0; k < p.topk; ++k) {
      const int id = p.ids[t * p.topk + k];
      if ((unsigned)id >= (unsigned)p.E) continue;
      int sum = 0;
      for (int w = 0; w < KW; ++w) sum += part[(k << kwshift) + w][tid];
      const float y = (float)sum * p.sd[(int64_t)id * p.H + n] * hs[k];
      out = __builtin_fmaf(p.weights[t * p.topk + k], y, out);
    }
    if (p.r) out += T::val(((const half_t*)p.r)[t * p.H + n]);
    ((half_t*)p.out)[t * p.H + n] = T::cvt1(out);
  }
}

// How a few tokens' second half is laid out; kw 0: it has no room.
struct TokenPlan {
  int kw, cols, xstride, bytes;
};
TokenPlan token_plan(int64_t T, int H, int F, int E, int topk, int num_cus) {
  TokenPlan l{};
  if (!few_tokens(T, E, topk) || topk > 16 || !own_bytes(1, H)) return l;
  int kw = 1;
  while (2 * kw * topk <= 16) kw *= 2;
  l.cols = (int64_t)H / 16 * T >= num_cus ? 16 : 8;
  l.xstride = (F + 255) / 256 * 256 + 64;
  l.bytes = topk * (kw * kTokenRing * kTokenSlot + l.xstride);
  if (F <= kw * 64 * 8 * kTokenPieces && l.bytes <= kRowsLds) l.kw = kw;
  return l;
}

// Rows of the tiles of both halves: 16 (the kernel for few rows) where an expert
// has fewer than 24 on average, else what takes least by the estimate, with half
// a tile more an expert for the last ones.  In us, both halves on 256 / on 128 /
// 256 and 128: 4,096 tokens, 2 of 8 experts of 2,048 x 8,192 584 / 612 / 568; 8 of
// 64 of 2,048 x 1,024 425 / 458 / 449; 512, 4 of 16 of 2,048 x 1,024 74 / 65 / 69.
struct ExpertsTiles {
  int up, down;
};
ExpertsTiles experts_tiles(int64_t P, int H, int F, int E, int num_cus) {
  if (P / E < 24) return {16, 16};
  auto best = [&](int N, int K, int sides) {
    int size = 0;
    float least = 0.f;
    for (int s : {256, 128, 64}) {
      const int64_t cols = s / sides, tiles = (P / s + E / 2 + 1) * ((N + cols - 1) / cols);
      float t = tile_time(s, tiles, (K + kChunk - 1) / kChunk, num_cus);
      if (s < 256) t += 4.f * (float)((tiles + num_cus - 1) / num_cus);  // the gather's way to a tile's first chunk
      if (size == 0 || t < least) size = s, least = t;
    }
    return size;
  };
  return {best(F, H, 2), best(H, F, 1)};
}

struct ExpertsLayout {
  ExpertsTiles size;
  int tile;  // of the plan: the larger one
  int64_t max_tiles, xq, xs, tiles, info, tok, pair, h, hq, hs, y, bytes;
};
ExpertsLayout experts_layout(int64_t T, int H, int F, int E, int topk, int num_cus) {
  ExpertsLayout l{};
  const int64_t P = T * topk;
  l.size = experts_tiles(P, H, F, E, num_cus);
  l.tile = l.size.up > l.size.down ? l.size.up : l.size.down;
  l.max_tiles = P / l.tile + (P < E ? P : E);
  auto take = [&](int64_t n) {
    const int64_t at = l.bytes;
    l.bytes += (n + 255) / 256 * 256;
    return at;
  };
  if (token_plan(T, H, F, E, topk, num_cus).kw) {
    l.h = take(P * F * 2);
    return l;
  }
  l.xq = take(T * H);
  l.xs = take(T * 4);
  l.tiles = take(l.max_tiles * (int64_t)sizeof(TileRec));
  l.info = take(8);
  l.tok = take(P * 4);
  l.pair = take(P * 4);
  l.h = take(P * F * 2);
  l.hq = take(P * F);
  l.hs = take(P * 4);
  l.y = take(P * H * 4);
  return l;
}

template <class T, int S, int MODE>
hipError_t experts_product(const I8Args& a, I8Group g, const ExpertsLayout& l, int size, int64_t pairs, int num_cus,
                           hipStream_t s) {
  if (size == 16) {
    const int64_t busy = pairs < g.experts ? pairs : g.experts;
    return rows_launch<T, S, MODE>(a, g, 1, l.max_tiles, busy, false, num_cus, s);
  }
  g.shift = __builtin_ctz(l.tile / size);
  return tile_launch<T, S, MODE>(a, g, l.max_tiles << g.shift, TilePlan{size, 1}, num_cus, s);
}

template <class T>
hipError_t experts_run(const ExpertsArgs& p, int num_cus, hipStream_t s) {
  const int64_t P = p.T * p.topk;
  const int64_t up_bytes = (int64_t)((p.F + 15) / 16) * ((p.H + 63) / 64) * 1024;
  const int64_t down_bytes = (int64_t)((p.H + 15) / 16) * ((p.F + 63) / 64) * 1024;
  const ExpertsLayout l = experts_layout(p.T, p.H, p.F, p.E, p.topk, num_cus);
  char* const ws = (char*)p.ws;
  const TokenPlan tp = token_plan(p.T, p.H, p.F, p.E, p.topk, num_cus);
  if (tp.kw) {
    const I8Group g{nullptr, nullptr, nullptr, nullptr, up_bytes, 0, p.ids, p.topk, p.E};
    const I8Args up{p.T, p.F, p.H, 2, p.x, nullptr, nullptr, {{p.wg, p.sg, nullptr}, {p.wu, p.su, nullptr}},
                    nullptr, p.act, ws + l.h, p.dtype, nullptr, nullptr};
    const hipError_t e = rows_launch<T, 2, UP>(up, g, 1, P, P, true, num_cus, s);
    if (e != hipSuccess) return e;
    const auto kern = tp.cols == 8 ? &i8_token_down_kernel<T, 8> : &i8_token_down_kernel<T, 16>;
    if (tp.bytes > 60 * 1024) {
      const hipError_t e2 = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, kRowsLds);
      if (e2 != hipSuccess) return e2;
    }
    hipLaunchKernelGGL(kern, dim3(p.H / tp.cols, (unsigned)p.T), dim3(p.topk * tp.kw * kWave), tp.bytes, s, p,
                       (const half_t*)(ws + l.h), down_bytes, __builtin_ctz(tp.kw), tp.xstride);
    return hipGetLastError();
  }
  I8Group g{(const TileRec*)(ws + l.tiles), (const int*)(ws + l.info), (const int*)(ws + l.tok), (const int*)(ws + l.pair), 0,
            0, p.ids, p.topk, p.E};
  const int wpr = p.H <= 2048 ? 1 : p.H <= 8192 ? 4 : 16;
  const auto plan = wpr == 1 ? &i8_plan_kernel<T, 1> : wpr == 4 ? &i8_plan_kernel<T, 4> : &i8_plan_kernel<T, 16>;
  hipLaunchKernelGGL(plan, dim3((unsigned)(p.E + (p.T + 16 / wpr - 1) / (16 / wpr))), dim3(1024), 0, s, p.ids, P, p.E, p.topk,
                     l.tile, (TileRec*)(ws + l.tiles), (int*)(ws + l.info), (int*)(ws + l.tok), (int*)(ws + l.pair),
                     (const half_t*)p.x, p.H, ws + l.xq, (float*)(ws + l.xs));
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  I8Args up{p.T, p.F, p.H, 2, nullptr, ws + l.xq, (const float*)(ws + l.xs), {{p.wg, p.sg, nullptr}, {p.wu, p.su, nullptr}},
            nullptr, p.act, ws + l.h, p.dtype, nullptr, nullptr};
  g.wbytes = up_bytes;
  if ((e = experts_product<T, 2, UP>(up, g, l, l.size.up, P, num_cus, s)) != hipSuccess) return e;
  if ((e = rows_to_bytes_launch<T>(ws + l.h, P, p.F, ws + l.hq, (float*)(ws + l.hs), s, g.info + 1)) != hipSuccess) return e;
  I8Args down{P, p.H, p.F, 1, nullptr, ws + l.hq, (const float*)(ws + l.hs), {{p.wd, p.sd, nullptr}, {}},
              nullptr, GP_ACT_NONE, ws + l.y, p.dtype, nullptr, nullptr};
  g.wbytes = down_bytes;
  if ((e = experts_product<F16, 1, DOWN>(down, g, l, l.size.down, P, num_cus, s)) != hipSuccess) return e;
  const int64_t pieces = p.T * (p.H / 8);
  hipLaunchKernelGGL((i8_combine_kernel<T>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, p, (const float*)(ws + l.y));
  return hipGetLastError();
}

}  // namespace

int64_t i8_workspace(int64_t M, int N, int K, bool x16, int sides, int num_cus) {
  return layout(M, N, K, x16, sides, num_cus).bytes;
}

int64_t i8_experts_workspace(int64_t T, int H, int F, int E, int topk, int num_cus) {
  return experts_layout(T, H, F, E, topk, num_cus).bytes;
}

hipError_t i8_experts_launch(const ExpertsArgs& a, int num_cus, hipStream_t s) {
  return a.dtype == GP_DTYPE_BF16 ? experts_run<BF16>(a, num_cus, s) : experts_run<F16>(a, num_cus, s);
}

hipError_t i8_launch(const I8Args& a, int num_cus, hipStream_t s) {
  if (a.dtype == GP_DTYPE_BF16) return a.sides == 2 ? launch<BF16, 2>(a, num_cus, s) : launch<BF16, 1>(a, num_cus, s);
  return a.sides == 2 ? launch<F16, 2>(a, num_cus, s) : launch<F16, 1>(a, num_cus, s);
}

}  // namespace gp
