// Products with 4-bit weights: out = act(x W + b) [or x W + b + r], and the
// gated pair act(x Wg + bg) * (x Wu + bu), W[k][n] = s[k / G][n] (q[k][n] - z[k / G][n]).
// No counterpart in the reference, whose GEMM stages take 16-bit weights
// (common/bulksync_gemm.cuh:13-110).
//
// Words.  Word [k / 8][n] holds q of eight consecutive k, the lowest in the low
// bits: eight k of one column are what one lane of an MFMA holds, so a word is
// a lane's operand, and the weights need no other layout than [K / 8, N].
//
// From a word to an operand.  A byte 0 .. 15 read as e4m3 is q 2^-9, denormal
// or not; a word masked, and a word >> 4 masked, are four such bytes each, and
// one conversion by 2^9 makes two of them q in 16 bits, exactly.  The operand
// holds the eight k in the order 0 2 4 6 1 3 5 7, and x is put in the same
// order.  Per group of G rows the matrix cores sum x q and, against a column of
// ones, x; then
//   sum x (q - z) = sum x q - z sum x
// in fp32, and times s into the running sum.  The weights are never rounded.
// s x (q - z) is so the difference of two that are up to 15 and |z| times s x,
// and an x leaves 2^-24 of those behind where its weight is small or zero.
// (64 + q and 128 + q, q put into a mantissa, are as many instructions, but
// leave 2^-24 of 64 to 150 times s x: an x 5,000 times as large as the others,
// its weights zero, then moves an fp16 result by more than its rounding does,
// and ten times as many results of 8,192 k differ from an fp32 product's.)
#include <hip/hip_runtime.h>
#include <type_traits>

#include "../../include/gpipes.h"
#include "gp_kernels.hpp"
#include "row_ops.hpp"

namespace gp {
namespace {

template <class T>
struct Q4;
template <>
struct Q4<F16> : F16 {
  // bytes 2 HI and 2 HI + 1 of u, each 0 .. 15
  template <bool HI>
  __device__ static unsigned bytes2(unsigned u) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 512.f, HI));
  }
  __device__ static f4 mma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  // s + both halves of u
  __device__ static float add2(unsigned u, float s) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, u), h2{(half_t)1.f, (half_t)1.f}, s, false);
  }
};
template <>
struct Q4<BF16> : BF16 {
  template <bool HI>
  __device__ static unsigned bytes2(unsigned u) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 512.f, HI));
  }
  __device__ static f4 mma16(h8 a, h8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  }
  __device__ static float add2(unsigned u, float s) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, u), bf2{(__bf16)1.f, (__bf16)1.f}, s, false);
  }
};

// The operand q of a word, k order 0 2 4 6 1 3 5 7.
template <class T>
__device__ __forceinline__ h8 q_operand(unsigned w) {
  const unsigned e = w & 0x0F0F0F0Fu, d = (w >> 4) & 0x0F0F0F0Fu;
  return __builtin_bit_cast(h8, u32x4{Q4<T>::template bytes2<false>(e), Q4<T>::template bytes2<true>(e),
                                      Q4<T>::template bytes2<false>(d), Q4<T>::template bytes2<true>(d)});
}

// Eight values of x in that order.
__device__ __forceinline__ h8 x_operand(u32x4 v) {
  u32x4 o;
  o[0] = __builtin_amdgcn_perm(v[1], v[0], 0x05040100u);
  o[1] = __builtin_amdgcn_perm(v[3], v[2], 0x05040100u);
  o[2] = __builtin_amdgcn_perm(v[1], v[0], 0x07060302u);
  o[3] = __builtin_amdgcn_perm(v[3], v[2], 0x07060302u);
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

// Eight neighbouring outputs of row m from column n (cnt of them inside the row).
template <class T>
__device__ __forceinline__ void q4_store8(const Q4Args& p, int64_t m, int n, int cnt, float (&v)[8],
                                          const float (&u)[8]) {
  float t[8];
  if (p.side[0].b) {
    load8<T>((const half_t*)p.side[0].b + n, cnt, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
  }
  apply_act8(v, p.act);
  if (p.sides == 2) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = 0.f;
    if (p.side[1].b) load8<T>((const half_t*)p.side[1].b + n, cnt, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= u[e] + t[e];
  }
  if (p.r) {
    load8<T>((const half_t*)p.r + m * p.N + n, cnt, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
  }
  store8<T>((half_t*)p.out + m * p.N + n, cnt, v);
}

// Workgroup b of n, renumbered so that neighbours in the result run on one XCD
// (b % 8): they read neighbouring columns, and 16 of them are half of a
// 128-byte line, which two XCDs would each fetch whole.
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int x = b & 7, i = b >> 3, q = n >> 3, rem = n & 7;
  return x * q + (x < rem ? x : rem) + i;
}

// v has its value here: the compiler does not put off what it comes from (two
// groups' sums at once would not fit the registers).
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }

constexpr int kChunk = 128;  // k that a wave takes at a time, the largest group
constexpr int kHalf = 64;    // k of a wave's one load: two MFMA steps

// The scales (or zeros) of CW neighbouring columns as they lie in memory.  A
// load that would pass the matrix's end begins CW values before it instead:
// only columns of its last row can then be misplaced, and shifted() puts them
// right.  No branch lies between the load and its first use.
template <int CW>
struct Cols {
  typedef unsigned short vec __attribute__((ext_vector_type(CW), aligned(2)));
  typedef typename std::conditional<CW == 4, unsigned long long, unsigned>::type bits;
  bits v;
  __device__ __forceinline__ void load(const unsigned short* m, int64_t at, int64_t last) {
    const unsigned short* p = m + (at < last ? at : last);
    if constexpr (CW == 1) v = *p;
    if constexpr (CW == 2) v = __builtin_bit_cast(unsigned, *(const vec*)p);
    if constexpr (CW == 4) v = __builtin_bit_cast(unsigned long long, *(const vec*)p);
  }
  __device__ __forceinline__ Cols shifted(int64_t at, int64_t last) const {
    Cols r = *this;
    if constexpr (CW > 1) r.v >>= at > last ? 16 * ((int)(at - last) & (CW - 1)) : 0;
    return r;
  }
  template <class T>
  __device__ __forceinline__ float val(int t) const {
    return T::val(__builtin_bit_cast(half_t, (unsigned short)(v >> (16 * t))));
  }
};

// ---------------------------------------------------------------------------
// Few rows: every wave of a workgroup multiplies its share of k with the
// workgroup's 16 CW columns of S weights, and the shares are joined through
// LDS in the order of the waves.  A workgroup reads all of x, from L2, which
// costs more than its words where rows are many; the two weights of a gated
// product share those reads.  Bound by a CU's loads (16 rows, 8,192 columns
// from 8,192 k: 10.8 us, 3.3 TB/s; a CU's 128 KiB of words would take 5 us at
// the 26 bytes a ns that it gets from the last cache, its 256 KiB of x 3.7 us
// at the 70 from L2, and the rest is the first loads' latency and the join).
// ---------------------------------------------------------------------------
// Waves of a workgroup at most: sixteen where a wave's tiles leave registers for
// them and k is worth it (20 rows, 4,096 columns from 16,384 k: 18.9 us, with
// eight 21.1; from 4,096 k 7.4 and 7.5; three tiles a wave, 37 rows, 4,093 columns from
// 4,072 k: 14.4 and 14.1).
constexpr int rows_waves(int tiles, int mt) { return mt == 1 || tiles * mt <= 2 ? 16 : 8; }

template <int CW, int S, int MT, int SG>
struct Half {
  unsigned w[2][S * CW];
  u32x4 x[2][MT];
  Cols<CW> s[S][SG], z[S][SG];
};

template <class T, int CW, int S, int MT, int G, bool FOUR>
__global__ __launch_bounds__(64 * rows_waves(CW * S, MT)) void q4_rows_kernel(Q4Args p) {
  constexpr int SG = G < kHalf ? kHalf / G : 1;  // groups a half (G 128: one every other half)
  constexpr int E = FOUR ? 1 : 4;                // accumulator elements that hold rows (FOUR: at most four rows)
  constexpr int COLS = 16 * CW, NT = S * CW;
  constexpr int TOK = FOUR ? 4 : 16;
  constexpr int PART = rows_waves(NT, MT) * TOK * COLS * S * 4, XS = FOUR ? 0 : rows_waves(NT, MT) * MT * 2048;
  __shared__ __attribute__((aligned(1024))) char lds[PART > XS ? PART : XS];
  const int lane = threadIdx.x & 63, j = lane & 15, lg = lane >> 4;
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int N = p.N, K = p.K;
  const int n0 = xcd_order(blockIdx.x, gridDim.x) * COLS;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const int rows = p.M - m0 < 16 * MT ? (int)(p.M - m0) : 16 * MT;
  const int groups = (K + G - 1) / G;
  const int chunks = (K + kChunk - 1) / kChunk;
  const auto wr0 = make_rsrc(p.side[0].wq, (int)((int64_t)K * N / 2));
  const auto wr1 = make_rsrc(p.side[S - 1].wq, (int)((int64_t)K * N / 2));
  const auto xr = make_rsrc((const half_t*)p.x + m0 * K, rows * K * 2);
  const int col = n0 + CW * j;
  const bool inside = n0 + COLS <= N;
  const int64_t last = (int64_t)groups * N - CW;
  // Row i of the x operand: row i, or with at most four rows row i / 4, which
  // lands in element 0 of the accumulators of the lanes of group i / 4.
  //
  // An operand takes 64 bytes of each of 16 rows, half a line, and a line whose
  // halves two instructions ask for is fetched twice from L2.  So eight lanes
  // load a row's 128 bytes of a half, and the rows turn into operands through a
  // piece of LDS that is the wave's own (16 rows, 8,192 columns from 8,192 k:
  // 13.4 us by halves of lines, 10.8 so; 64 rows, 4,096 from 4,096: 20 and 13).
  // 16-byte piece c of a row lies there at c ^ row % 8.
  char* const xs = lds + (FOUR ? 0 : wave * (MT * 2048));
  const int xrow = FOUR ? j >> 2 : lane >> 3;

  // half t of this wave: chunks wave, wave + waves, ..., two halves each
  auto load = [&](int t, Half<CW, S, MT, SG>& q, bool second) {
    const int k0 = (wave + (t >> 1) * waves) * kChunk + (second ? kHalf : 0);
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int k = k0 + st * 32 + lg * 8;
      // past the weight's end and past the rows' end (and the last row) nothing is read: zeros, and a zero of x is
      // what no word can make count
      const unsigned off = k < K ? ((unsigned)(k >> 3) * (unsigned)N + (unsigned)col) * 4u : 0xFFFFFFE0u;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const auto wr = s ? wr1 : wr0;
        unsigned* w = q.w[st] + s * CW;
        if constexpr (CW == 4) {
          const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(wr, (int)off, 0, 0);
          w[0] = v[0], w[1] = v[1], w[2] = v[2], w[3] = v[3];
        } else if constexpr (CW == 2) {
          const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(wr, (int)off, 0, 0);
          w[0] = v[0], w[1] = v[1];
        } else {
          w[0] = __builtin_amdgcn_raw_buffer_load_b32(wr, (int)off, 0, 0);
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int xk = FOUR ? k : k0 + (lane & 7) * 8;
        const int xo = ((FOUR ? xrow : mt * 16 + st * 8 + xrow) * K + xk) * 2;
        q.x[st][mt] = __builtin_amdgcn_raw_buffer_load_b128(xr, xk < K ? xo : 0x7FFFFFE0, 0, 0);
      }
    }
    if (G < kChunk || second) {
#pragma unroll
      for (int g = 0; g < SG; ++g) {
        int gi = k0 / G + g;
        gi = gi < groups ? gi : groups - 1;
        const int64_t at = (int64_t)gi * N + col;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const Q4Side& sd = p.side[s];
          q.s[s][g].load((const unsigned short*)sd.s, at, last);
          q.z[s][g].load((const unsigned short*)(sd.z ? sd.z : sd.s), at, last);
        }
      }
    }
  };

  float tot[NT][MT][E] = {};
  f4 acc[NT][MT], sum[MT];
  const h8 ones = __builtin_bit_cast(h8, u32x4{T::kOne * 0x10001u, T::kOne * 0x10001u, T::kOne * 0x10001u,
                                               T::kOne * 0x10001u});
  auto mul = [&](int h, const Half<CW, S, MT, SG>& q, bool second) {
    if constexpr (!FOUR) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int st = 0; st < 2; ++st)
          *(h8*)(xs + mt * 2048 + (st * 8 + xrow) * 128 + (((lane & 7) ^ xrow) << 4)) = x_operand(q.x[st][mt]);
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int k = (second ? kHalf : 0) + st * 32;
      if (k % G == 0) {  // a group begins
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          sum[mt] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][mt] = f4{0.f, 0.f, 0.f, 0.f};
        }
      }
      h8 b[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) b[t] = q_operand<T>(q.w[st][t]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        h8 a;
        if constexpr (FOUR) {
          a = x_operand(q.x[st][mt]);
        } else {
          a = *(const h8*)(xs + mt * 2048 + j * 128 + (((st * 4 + lg) ^ (j & 7)) << 4));
        }
        sum[mt] = Q4<T>::mma16(a, ones, sum[mt]);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][mt] = Q4<T>::mma16(a, b[t], acc[t][mt]);
      }
      if ((k + 32) % G == 0) {  // and ends
        const int g = G < kHalf ? st : 0;
#pragma unroll
        for (int sd = 0; sd < S; ++sd) {
          Cols<CW> qs = q.s[sd][g], qz = q.z[sd][g];
          if (!inside) {
            int gi = (wave + (h >> 1) * waves) * (kChunk / G) + k / G;
            gi = gi < groups ? gi : groups - 1;
            const int64_t at = (int64_t)gi * N + col;
            qs = qs.shifted(at, last), qz = qz.shifted(at, last);
          }
#pragma unroll
          for (int t = 0; t < CW; ++t) {
            const float s = qs.template val<T>(t);
            const float z = p.side[sd].z ? qz.template val<T>(t) : 8.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int e = 0; e < E; ++e) {
                float& v = tot[sd * CW + t][mt][e];
                v = __builtin_fmaf(s, __builtin_fmaf(-z, sum[mt][e], acc[sd * CW + t][mt][e]), v);
                pin(v);
              }
          }
        }
      }
      // steps are not mixed: the compiler would spread their operands over more registers than there are
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Two halves in flight, a chunk (four are slower: 16 rows, 1,024 columns from
  // 1,024 k 3.3 us and 4.2, 4,096 from 16,384 13.4 and 14.0).  Loads are issued
  // without a condition, so that the compiler counts them: those past the wave's
  // last chunk read nothing.
  const int halves = wave < chunks ? 2 * ((chunks - 1 - wave) / waves + 1) : 0;
  Half<CW, S, MT, SG> q[2];
  if (halves) {
#pragma unroll
    for (int i = 0; i < 2; ++i) load(i, q[i], i & 1);
    for (int t = 0; t < halves; t += 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mul(t + i, q[i], i & 1);
        load(t + 2 + i, q[i], i & 1);
      }
    }
  }

  float* const part = (float*)lds;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (mt || !FOUR) __syncthreads();  // every wave is done with what lies there
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int t = 0; t < NT; ++t)
        part[((wave * TOK + (FOUR ? lg : 4 * lg + e)) * S + t / CW) * COLS + CW * j + t % CW] = tot[t][mt][e];
    __syncthreads();
    for (int i = threadIdx.x; i < TOK * COLS; i += blockDim.x) {
      const int tok = i / COLS, row = mt * 16 + tok, n = i % COLS;
      if (row >= rows || n0 + n >= N) continue;
      float v = 0.f, u = 0.f;
      for (int w = 0; w < waves; ++w) {
        v += part[(w * TOK + tok) * S * COLS + n];
        if (S == 2) u += part[((w * TOK + tok) * S + 1) * COLS + n];
      }
      q4_store<T>(p, m0 + row, n0 + n, v, u);
    }
  }
}

// ---------------------------------------------------------------------------
// One token.  Words come faster than 16-bit operands can be made
// of them (seven operations a word), so here the operands are 8 bits: a byte
// 0 .. 15 read as e4m3 is q 2^-9, denormal or not, and a word is two dwords of
// such bytes, w and w >> 4 masked -- k in the order 0 2 4 6, 1 3 5 7.  x, in
// chunks of 128 k, is written with six signed digits to the base 32, each a
// whole number up to 16 that e4m3 holds: x = 2^e (d0 + d1 / 32 + ... + d5 /
// 32^5), 2^e such that the chunk's largest value has d0 in [8, 16].  That is x
// to 2^-29 of the chunk's largest, a 32nd of what an fp32 sum keeps of it: a
// value 10,000 times as large as its neighbours, its weights zero, leaves
// nothing behind that a result shows.  (With four digits, 2^-19, such a value
// made twenty times an fp16 result's rounding, with five a tenth of it more.)
//
// Whole numbers, because the 8-bit MFMAs add their products with fewer bits
// than fp32: of products far apart in size they lose what is 2^-14 of the
// largest (measured).  Those of a digit with q are whole and at most 240, so
// nothing is lost, and the six digits' sums are added in fp32.
//
// Digit p is row p of the MFMA (16 x 16 x 128, whose scale operand brings 2^e /
// 32^p).  Each row has its own running sum, and the six are added at the end.
// A group shorter than 128 has an MFMA of its own, where the other blocks of
// the weight go under 2^-127.
//
// Such a call is over in the time of a few memory latencies, and code that no
// wave has run yet is fetched from memory too.  So all that the workgroup will
// read is asked for first: x, the scales and kRing chunks of every wave's
// words, the latter by copies into LDS that hold no registers; and the code
// is short (rolled loops, no copy of it for a size of group).  2 x 16,384 columns
// from 4,096 k: 13.5 us, 5.2 TB/s; 4,096 columns from 16,384 k: 10.1 us, 3.5
// TB/s, of which 5 are the words and 3 the digits of x, that every workgroup
// makes for itself; 1,024 from 1,024: 3.2 us, the latencies of a launch, two
// loads and the join.  Rings of four to eight chunks were slower (more LDS to
// hand out, later first words).
// ---------------------------------------------------------------------------
constexpr int kTokenCols = 16;
constexpr int kDigits = 6;
constexpr int kRing = 2;  // chunks of 1 KiB that a wave has in flight
constexpr int kTokenLds = 158 * 1024;  // of dynamic LDS at most: a CU's 160 KiB less 2 for the waves' sums

// LDS, in this order: x's digits, rows of K bytes 16 bytes apart in banks; the
// powers, a byte a chunk; every wave's ring; every wave's scales and zeros, 32
// bytes a group, in copies of 256.
struct TokenLds {
  int xstride, powers, ring, scales, wave_scales, bytes;
};
inline TokenLds token_lds(int K, int group, int waves, int kw, bool z) {
  TokenLds l;
  const int chunks = (K + kChunk - 1) / kChunk, cpw = (chunks + kw - 1) / kw;
  l.xstride = (chunks * kChunk + 255) / 256 * 256 + 16;
  l.powers = kDigits * l.xstride;
  l.ring = (l.powers + chunks + 1023) / 1024 * 1024;
  l.scales = l.ring + waves * kRing * 1024;
  l.wave_scales = (cpw * (kChunk / group) + 7) / 8 * 256;
  l.bytes = l.scales + waves * l.wave_scales * (z ? 2 : 1);
  return l;
}

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Eight values of x, a sixteenth of a chunk (the others are in the lanes of
// this row of sixteen): their digits to LDS rows 0 .. 5, the chunk's power.
template <class T>
__device__ __forceinline__ void put_digits(u32x4 v, GP_LDS char* at, int xstride, GP_LDS char* power, bool first) {
  float x[8];
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = T::val(__builtin_bit_cast(half_t, (unsigned short)(v[e] & 0xFFFF)));
    x[2 * e + 1] = T::val(__builtin_bit_cast(half_t, (unsigned short)(v[e] >> 16)));
    // the maximum drops a NaN, which stays one in its own digits
    top = fmaxf(top, fmaxf(fabsf(x[2 * e]), fabsf(x[2 * e + 1])));
  }
#define GP_DPP_F(v, ctrl) __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), ctrl, 0xF, 0xF, false))
  top = fmaxf(top, GP_DPP_F(top, 0x128));  // row_ror:8
  top = fmaxf(top, GP_DPP_F(top, 0x124));  // row_ror:4
  top = fmaxf(top, GP_DPP_F(top, 0x4E));
  top = fmaxf(top, GP_DPP_F(top, 0xB1));
#undef GP_DPP_F
  // e, biased; not so small that the last digit's power would pass zero
  int e = (__builtin_bit_cast(int, top) >> 23) - 3;
  e = e < 25 ? 25 : e;
  const float up = __builtin_bit_cast(float, (254 - e) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= up;
#pragma unroll
  for (int p = 0; p < kDigits; ++p) {
    float d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      d[i] = __builtin_rintf(x[i]);
      x[i] = (x[i] - d[i]) * 32.f;  // exact: at most 16
    }
    u32x2 o;
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // even k, odd k
      const int w = __builtin_amdgcn_cvt_pk_fp8_f32(d[h], d[2 + h], 0, false);
      o[h] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(d[4 + h], d[6 + h], w, true);
    }
    *(GP_LDS u32x2*)(at + p * xstride) = o;
  }
  if (first) *power = (char)e;
}

// CT: tiles of 16 columns a workgroup; KW: waves along k.  Wave
// (side CT + ct) KW + kw takes chunks [kw cpw, (kw + 1) cpw) of column tile ct
// of weight `side`.
template <class T>
__global__ __launch_bounds__(1024) void q4_token_kernel(Q4Args p, int ctshift, int kwshift, int gshift, TokenLds l) {
  __shared__ float part[16][2][kTokenCols];  // of a wave: the first four digits' sums, the last two's
  GP_LDS char* lds = dyn_lds();
  const int CT = 1 << ctshift, KW = 1 << kwshift;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, lg = lane >> 4;
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = wave & (KW - 1), tile = wave >> kwshift, ct = tile & (CT - 1), side = tile >> ctshift;
  const int N = p.N, K = p.K;
  const int n0 = xcd_order(blockIdx.x, gridDim.x) * (kTokenCols * CT);
  const int chunks = (K + kChunk - 1) / kChunk, cpw = (chunks + KW - 1) >> kwshift;
  const int c0 = kw * cpw, nc = chunks - c0 < cpw ? chunks - c0 : cpw;  // may be 0 or less: nothing
  const Q4Side sd = side ? p.side[1] : p.side[0];
  const int tcol = n0 + ct * kTokenCols;  // the tile's first column

  // Reads past the end of x's row, of the weight or of the scales bring zeros:
  // a zero of x is what no word can make count.
  // Scales: eight groups of 16 columns a copy, two columns a lane (N is even here).
  GP_LDS char* sl = lds + l.scales + wave * l.wave_scales;
  GP_LDS char* zl = sd.z ? sl + waves * l.wave_scales : sl;
  const int g0 = (c0 * kChunk) >> gshift, gbytes = ((K + (1 << gshift) - 1) >> gshift) * N * 2;
  const auto sr = make_rsrc(sd.s, gbytes), zr = make_rsrc(sd.z, gbytes);
#pragma unroll 1
  for (int i = 0; i < l.wave_scales / 256; ++i) {
    const int off = ((g0 + i * 8 + (lane >> 3)) * N + tcol + 2 * (lane & 7)) * 2;
    dma4_buf(sr, off, sl + i * 256);
    if (sd.z) dma4_buf(zr, off, zl + i * 256);
  }
  // x: a thread has eight k, and the conversion waits for them
  const int kend = chunks * kChunk;
  const auto xr = make_rsrc(p.x, K * 2);
  u32x4 xv = __builtin_amdgcn_raw_buffer_load_b128(xr, tid * 16, 0, 0);
  // A chunk's copy: 16 word rows of 16 columns, 16 bytes a lane.  A lane of the
  // MFMA's group lg holds k 16 lg .. + 15 of the chunk and of its second half,
  // so its words are rows 2 lg, 2 lg + 1, 8 + 2 lg, 9 + 2 lg; word i of group lg
  // lies at place 4 i + lg, where a wave's read of word i is 256 bytes in a row.
  const auto wr = make_rsrc(sd.wq, (int)((int64_t)K * N / 2));
  GP_LDS char* ring = lds + l.ring + wave * (kRing * 1024);
  const int wrow = 2 * ((lane >> 2) & 3) + ((lane >> 4) & 1) + 8 * (lane >> 5);
  unsigned woff = ((unsigned)(c0 * (kChunk / 8) + wrow) * (unsigned)N + (unsigned)(tcol + 4 * (lane & 3))) * 4u;
  const unsigned wstep = (unsigned)N * (kChunk / 8 * 4);
#pragma unroll
  for (int i = 0; i < kRing; ++i, woff += wstep) dma16_buf(wr, (int)(i < nc ? woff : 0xFFFFFFE0u), ring + i * 1024);
  wait_vmcnt<kRing>();  // this wave's scales, and its first part of x
  auto put = [&](int k) {
    if (k < kend)  // rows of sixteen threads, a chunk each
      put_digits<T>(xv, lds + k, l.xstride, lds + l.powers + k / kChunk, !(tid & 15));
  };
  put(tid * 8);
#pragma unroll 1
  for (int k = (blockDim.x + tid) * 8; k - tid * 8 < kend; k += blockDim.x * 8) {
    xv = __builtin_amdgcn_raw_buffer_load_b128(xr, k * 2, 0, 0);
    put(k);
  }
  lds_barrier();

  // Row j of the A operand: digit j (behind the last the last one's again, whose sums go unread).
  const int digit = j < kDigits ? j : kDigits - 1;
  GP_LDS const char* xl = lds + digit * l.xstride + c0 * kChunk + lg * 16;
  GP_LDS const char* pl = lds + l.powers + c0;
  const i32x8 one = {0x01010101, 0x01010101, 0x01010101, 0x01010101, 0x01010101, 0x01010101, 0x01010101, 0x01010101};
  const int ng = kChunk >> gshift, gb = (lg * 32) >> gshift;  // groups a chunk; the one of block lg, whose power this lane gives
  f4 tot = {0.f, 0.f, 0.f, 0.f};
  int at = 0;
#pragma unroll 1
  for (int t = 0; t < nc; ++t) {
    wait_vmcnt<kRing - 1>();
    GP_LDS char* slot = ring + at * 1024;
    at = at + 1 == kRing ? 0 : at + 1;
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *(GP_LDS const unsigned*)(slot + i * 256 + lg * 64 + j * 4);
    const u32x4 a0 = *(GP_LDS const u32x4*)(xl + t * kChunk), a1 = *(GP_LDS const u32x4*)(xl + t * kChunk + 64);
    const int pw = (int)*(GP_LDS const unsigned char*)(pl + t) - 5 * digit;
    // what was read is in registers before the slot takes the chunk kRing further on
    compiler_fence();
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    dma16_buf(wr, (int)(t + kRing < nc ? woff : 0xFFFFFFE0u), slot);
    woff += wstep;
    i32x8 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = (int)a0[i], a[4 + i] = (int)a1[i];
      b[2 * i] = (int)(w[i] & 0x0F0F0F0Fu), b[2 * i + 1] = (int)((w[i] >> 4) & 0x0F0F0F0Fu);
    }
#pragma unroll 1
    for (int g = 0; g < ng; ++g) {
      const f4 zero = {0.f, 0.f, 0.f, 0.f};
      const int wp = gb == g ? 127 + 9 : 0;
      const f4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, pw, 0, wp);
      const f4 sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, one, zero, 0, 0, 0, pw, 0, wp);
      const int sat = (t * ng + g) * 32 + j * 2;
      const float s = T::val(*(GP_LDS const half_t*)(sl + sat));
      const float zv = T::val(*(GP_LDS const half_t*)(zl + sat)), z = sd.z ? zv : 8.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) tot[e] = __builtin_fmaf(s, __builtin_fmaf(-z, sum[e], d[e]), tot[e]);
    }
  }

  // the waves of a column tile in their order
  if (lg < 2) part[wave][lg][j] = lg ? tot[0] + tot[1] : (tot[0] + tot[1]) + (tot[2] + tot[3]);
  __syncthreads();
  const int n = tid & (kTokenCols - 1), tl = tid / kTokenCols;
  if (tl < CT && n0 + tl * kTokenCols + n < N) {
    float v = 0.f, u = 0.f;
    auto sum = [&](int w) { return part[w][0][n] + part[w][1][n]; };
    for (int w = 0; w < KW; ++w) v += sum(tl * KW + w);
    if (p.sides == 2)
      for (int w = 0; w < KW; ++w) u += sum((CT + tl) * KW + w);
    q4_store<T>(p, 0, n0 + tl * kTokenCols + n, v, u);
  }
}

template <class T>
hipError_t token_launch(const Q4Args& a, int waves, int ct, int kw, const TokenLds& l, hipStream_t s) {
  const auto kern = &q4_token_kernel<T>;
  if (l.bytes > 60 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, kTokenLds);
    if (e != hipSuccess) return e;
  }
  const int cols = kTokenCols * ct;
  const int gshift = a.group == 32 ? 5 : a.group == 64 ? 6 : 7;
  hipLaunchKernelGGL(kern, dim3((unsigned)((a.N + cols - 1) / cols)), dim3(waves * kWave), l.bytes, s, a,
                     __builtin_ctz(ct), __builtin_ctz(kw), gshift, l);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of four waves computes 64 rows of 64 CW columns, a
// wave 16 CW of them.  x goes through LDS, in the operands' order, with its
// groups' sums; a wave takes its words from memory itself and makes operands
// of each once for its four row tiles.  With two weights two waves take each,
// the same 32 CW columns of both.  Where tiles are few, several workgroups share
// one, each with a part of k, leave their sums in a workspace in fp32, and a
// second kernel adds them in order.
//
// Bound by instruction issue: two waves a SIMD run about 430 instructions a
// chunk for 64 MFMAs (64 conversions, 48 masks and shifts for them, 64 fused
// multiply-adds of the groups' ends), the matrix cores busy 43% of the time and
// the vector units 61%.  4,096 rows, 4,096 columns from 4,096 k: 138 to 144 us, 0.95
// to 0.99 PFLOP/s (this card's library product of 16-bit operands of that size: 127).
// Tried and no faster: operands one to four steps ahead, words copied to LDS
// two chunks ahead, MFMAs and operand instructions interleaved by the scheduler's
// groups (163), wave priorities, offsets in scalar registers.
// ---------------------------------------------------------------------------
constexpr int kTileRows = 64;

// Sum of eight 16-bit values.
template <class T>
__device__ __forceinline__ float sum8(h8 v) {
  const u32x4 u = __builtin_bit_cast(u32x4, v);
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) s = Q4<T>::add2(u[e], s);
  return s;
}

// v + (v of the lane that the DPP control names), within sixteen lanes.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

template <class T, int CW, int G, bool Z>
__global__ __launch_bounds__(256, 2) void q4_tile_kernel(Q4Args p, int mtiles, int ntiles, float* ws) {
  constexpr int MT = 4, ROWS = kTileRows;
  constexpr int GPC = kChunk / G;  // groups a chunk
  constexpr int SPG = G / 32;      // MFMA steps a group
  __shared__ __attribute__((aligned(1024))) struct {
    char x[2][ROWS * kChunk * 2];
    float s[2][GPC][ROWS];
  } lds;
  auto& xs = lds.x;
  auto& ss = lds.s;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int N = p.N, K = p.K;
  // Neighbours of one XCD take eight row tiles of a column tile, then of the
  // next: 64 of them read eight tiles of x and eight of the weight.
  const int id = xcd_order(blockIdx.x, gridDim.x);
  const int gm0 = id / (8 * ntiles) * 8, rest = id % (8 * ntiles);
  const int gm = mtiles - gm0 < 8 ? mtiles - gm0 : 8;
  const int side = p.sides == 2 ? wave >> 1 : 0;
  const int64_t m0 = (int64_t)(gm0 + rest % gm) * ROWS;
  const int wcols = 64 * CW / p.sides;
  const int n0 = rest / gm * wcols, wn0 = n0 + (p.sides == 2 ? wave & 1 : wave) * (16 * CW);
  const int col = wn0 + CW * j;
  const int rows = p.M - m0 < ROWS ? (int)(p.M - m0) : ROWS;
  const int groups = (K + G - 1) / G, chunks = (K + kChunk - 1) / kChunk;
  const Q4Side sd = side ? p.side[1] : p.side[0];
  const auto wr = make_rsrc(sd.wq, (int)((int64_t)K * N / 2));
  const auto xr = make_rsrc((const half_t*)p.x + m0 * K, rows * K * 2);
  const unsigned short* sp = (const unsigned short*)sd.s;
  const unsigned short* zp = (const unsigned short*)(sd.z ? sd.z : sd.s);
  const bool inside = wn0 + 16 * CW <= N;
  const int64_t last = (int64_t)groups * N - CW;

  // this thread's part of a chunk of x: eight k of rows tid / 16 + 16 q
  const int xk = (tid & 15) * 8, xrow = tid >> 4;
  u32x4 xv[MT];
  auto load_x = [&](int c) {
    const int k = c * kChunk + xk;
#pragma unroll
    for (int q = 0; q < MT; ++q)
      xv[q] = __builtin_amdgcn_raw_buffer_load_b128(xr, k < K ? ((xrow + 16 * q) * K + k) * 2 : 0x7FFFFFE0, 0, 0);
  };
  // 16-byte piece c of a row lies at c ^ row % 16: sixteen rows' reads of one piece fall into different banks
  auto put_x = [&](int buf) {
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const int row = xrow + 16 * q;
      const h8 v = x_operand(xv[q]);
      *(h8*)(xs[buf] + row * (kChunk * 2) + (((tid & 15) ^ (row & 15)) << 4)) = v;
      float s = sum8<T>(v);
      s = add_dpp<0xB1>(s);                           // quad_perm [1,0,3,2]
      s = add_dpp<0x4E>(s);                           // quad_perm [2,3,0,1]
      if constexpr (G >= 64) s = add_dpp<0x141>(s);   // row_half_mirror
      if constexpr (G >= 128) s = add_dpp<0x140>(s);  // row_mirror
      ss[buf][(tid & 15) / (G / 8)][row] = Z ? -s : -8.f * s;  // the same from each lane of the group
    }
  };
  unsigned w[4][CW];
  Cols<CW> qs[GPC], qz[GPC];
  auto load_w = [&](int c, int st) {
    const unsigned off = ((unsigned)(c * (kChunk / 8) + st * 4 + lg) * (unsigned)N + (unsigned)col) * 4u;
    if constexpr (CW == 4) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(wr, (int)off, 0, 0);
      w[st][0] = v[0], w[st][1] = v[1], w[st][2] = v[2], w[st][3] = v[3];
    } else if constexpr (CW == 2) {
      const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(wr, (int)off, 0, 0);
      w[st][0] = v[0], w[st][1] = v[1];
    } else {
      w[st][0] = __builtin_amdgcn_raw_buffer_load_b32(wr, (int)off, 0, 0);
    }
  };
  auto group_at = [&](int c, int g) {
    const int gi = c * GPC + g < groups ? c * GPC + g : groups - 1;
    return (int64_t)gi * N + col;
  };
  auto load_s = [&](int c, int g) {
    qs[g].load(sp, group_at(c, g), last);
    if constexpr (Z) qz[g].load(zp, group_at(c, g), last);
  };

  float tot[CW][MT][4] = {};
  // One chunk.  Registers hold one chunk's words and scales, and each is asked
  // for again, a chunk ahead, when it has been used; the next chunk's x, which
  // was asked for a chunk ago, goes to the other buffer.
  auto chunk = [&](int c, int buf) {
    if (!inside) {
#pragma unroll
      for (int g = 0; g < GPC; ++g) {
        qs[g] = qs[g].shifted(group_at(c, g), last);
        if constexpr (Z) qz[g] = qz[g].shifted(group_at(c, g), last);
      }
    }
    h8 b[CW];
#pragma unroll
    for (int t = 0; t < CW; ++t) b[t] = q_operand<T>(w[0][t]);
    load_w(c + 1, 0);
    f4 acc[CW][MT];
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      const int g = st / SPG;
      h8 bn[CW];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const h8 x = *(const h8*)(xs[buf] + (mt * 16 + j) * (kChunk * 2) + (((st * 4 + lg) ^ j) << 4));
        if (st % SPG == 0) {
          // a group's sum begins at -z times that of x
          const f4 m = *(const f4*)&ss[buf][g][mt * 16 + 4 * lg];
#pragma unroll
          for (int t = 0; t < CW; ++t) {
            const float z = sd.z ? qz[g].template val<T>(t) : 8.f;
            acc[t][mt] = Q4<T>::mma16(x, b[t], Z ? f4{z * m[0], z * m[1], z * m[2], z * m[3]} : m);
          }
        } else {
#pragma unroll
          for (int t = 0; t < CW; ++t) acc[t][mt] = Q4<T>::mma16(x, b[t], acc[t][mt]);
        }
        if (st < 3) {
#pragma unroll
          for (int t = mt * CW / MT; t < (mt + 1) * CW / MT; ++t) bn[t] = q_operand<T>(w[st < 3 ? st + 1 : 3][t]);
        }
        if ((st + 1) % SPG == 0) {
#pragma unroll
          for (int t = 0; t < CW; ++t) {
            const float s = qs[g].template val<T>(t);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              tot[t][mt][e] = __builtin_fmaf(s, acc[t][mt][e], tot[t][mt][e]);
              pin(tot[t][mt][e]);
            }
          }
        }
      }
      if (st < 3) {
        load_w(c + 1, st + 1);
#pragma unroll
        for (int t = 0; t < CW; ++t) b[t] = bn[t];
      }
      if ((st + 1) % SPG == 0) load_s(c + 1, g);
    }
    put_x(buf ^ 1);
    load_x(c + 2);
    lds_barrier();
  };
  // this workgroup's part of k: all of it, or gridDim.y-th
  const int per = (chunks + gridDim.y - 1) / gridDim.y, c0 = blockIdx.y * per, c1 = c0 + per < chunks ? c0 + per : chunks;
  load_x(c0);
#pragma unroll
  for (int st = 0; st < 4; ++st) load_w(c0, st);
#pragma unroll
  for (int g = 0; g < GPC; ++g) load_s(c0, g);
  put_x(0);
  load_x(c0 + 1);
  lds_barrier();
#pragma unroll 1
  for (int c = c0; c < c1; c += 2) {
    chunk(c, 0);
    if (c + 1 >= c1) break;
    chunk(c + 1, 1);
  }

  if (gridDim.y > 1) {
    typedef float vec __attribute__((ext_vector_type(CW), aligned(4)));
    float* part = ws + ((int64_t)blockIdx.y * p.sides + side) * p.M * N;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = mt * 16 + 4 * lg + e;
        float* at = part + (m0 + row) * N + col;
        if (row < rows && col + CW <= N) {
          vec v;
          if constexpr (CW == 1) v = tot[0][mt][e];
          else
#pragma unroll
            for (int t = 0; t < CW; ++t) v[t] = tot[t][mt][e];
          *(vec*)at = v;
        } else if (row < rows) {
#pragma unroll
          for (int t = 0; t < CW - 1; ++t)
            if (col + t < N) at[t] = tot[t][mt][e];
        }
      }
    return;
  }

  // Out through LDS, half of the rows at a time: eight columns a thread, whole
  // lines a wave, and the epilogue's code once.  Of two weights the columns lie
  // side by side.
  constexpr int LD = 64 * CW + 4;
  static_assert((ROWS / 2) * LD * 4 <= (int)sizeof(lds), "half a tile fits x's buffers");
  float* tile = (float*)&lds;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    auto put = [&](int mt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float* at = tile + ((mt % (MT / 2)) * 16 + 4 * lg + e) * LD + wave * (16 * CW) + CW * j;
#pragma unroll
        for (int t = 0; t < CW; ++t) at[t] = tot[t][mt][e];
      }
    };
#pragma unroll
    for (int mt = 0; mt < MT / 2; ++mt) {
      if (half) {
        put(MT / 2 + mt);
      } else {
        put(mt);
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < (ROWS / 2) * (wcols / 8); i += 256) {
      const int row = i / (wcols / 8), n = i % (wcols / 8) * 8;
      if (half * (ROWS / 2) + row >= rows || n0 + n >= N) continue;
      float v[8], u[8];
      const float* at = tile + row * LD + n;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = at[e], u[e] = p.sides == 2 ? at[wcols + e] : 0.f;
      q4_store8<T>(p, m0 + half * (ROWS / 2) + row, n0 + n, N - n0 - n, v, u);
    }
    __syncthreads();
  }
}

// The parts of k added in order, and the epilogue: eight columns of a row a thread.
template <class T>
__global__ __launch_bounds__(256) void q4_join_kernel(Q4Args p, const float* ws, int parts) {
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  const int pieces = (p.N + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.M * pieces) return;
  const int64_t m = i / pieces;
  const int n = (int)(i - m * pieces) * 8, cnt = p.N - n;
  float v[2][8] = {};
#pragma unroll 4
  for (int k = 0; k < parts; ++k)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= p.sides) continue;
      const float* at = ws + (((int64_t)k * p.sides + s) * p.M + m) * p.N + n;
      if (cnt >= 8) {
        const f4u a = *(const f4u*)at, b = *(const f4u*)(at + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[s][e] += a[e], v[s][4 + e] += b[e];
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (e < cnt) v[s][e] += at[e];
      }
    }
  q4_store8<T>(p, m, n, cnt, v[0], v[1]);
}

// How a product on tiles is cut: columns of a tile (64 CW) and parts of k.
struct TilePlan {
  int cw, parts;
};
// The least of an estimate in us.  A chunk takes a workgroup `alone` by itself
// on its CU and `shared` in company (4096 k are 32 chunks: 64 rows of 4,096
// columns 50, 37 and 30 us with CW 4, 2 and 1; 1,024 rows, which are one, two and
// four workgroups a CU, 52, 53 and 63); the second kernel takes 3 us and the
// workspace's way to memory and back.  128 rows of 4,096 columns from 4,096 k:
// 64 columns a tile and three parts 19 us, 256 columns in one part 50.  Not in it:
// a tile's prologue and epilogue, a third of the time at 1,024 k, and the group
// and zeros (all of the above: groups of 128 without zeros).
TilePlan tile_plan(int64_t M, int N, int K, int sides, int num_cus) {
  const int64_t mtiles = (M + kTileRows - 1) / kTileRows;
  const int chunks = (K + kChunk - 1) / kChunk;
  TilePlan best{4, 1};
  float least = 0.f;
  for (int cw = 4; cw >= 1; cw /= 2) {
    const int64_t cols = 64 * cw / sides, tiles = mtiles * ((N + cols - 1) / cols);
    const float alone = cw == 4 ? 1.5f : cw == 2 ? 1.1f : 0.85f, shared = cw == 4 ? 1.25f : cw == 2 ? 0.8f : 0.47f;
    for (int parts = 1; parts <= 16 && parts <= chunks; ++parts) {
      const float per_cu = (float)((tiles * parts + num_cus - 1) / num_cus);
      const float turn = shared * per_cu > alone ? shared * per_cu : alone;
      float t = (float)((chunks + parts - 1) / parts) * turn;
      if (parts > 1) t += 3.f + (float)parts * (float)M * (float)N * (float)sides * 8.f / 4e6f;
      if (least == 0.f || t < least) best = TilePlan{cw, parts}, least = t;
    }
  }
  return best;
}

template <class T, int CW>
hipError_t tile_launch(const Q4Args& a, int parts, hipStream_t s) {
  const int64_t mtiles = (a.M + kTileRows - 1) / kTileRows, cols = 64 * CW / a.sides;
  const int64_t ntiles = (a.N + cols - 1) / cols;
  if (mtiles * ntiles > (int64_t(1) << 31) - 1) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(mtiles * ntiles), (unsigned)parts), block(256);
  const bool z = a.side[0].z || a.side[1].z;
  float* ws = (float*)a.ws;
#define GP_CASE(g)                                                                                                \
  case g:                                                                                                         \
    if (z)                                                                                                        \
      hipLaunchKernelGGL((q4_tile_kernel<T, CW, g, true>), grid, block, 0, s, a, (int)mtiles, (int)ntiles, ws);   \
    else                                                                                                          \
      hipLaunchKernelGGL((q4_tile_kernel<T, CW, g, false>), grid, block, 0, s, a, (int)mtiles, (int)ntiles, ws);  \
    break;
  switch (a.group) {
    GP_CASE(32) GP_CASE(64) GP_CASE(128)
    default: return hipErrorInvalidValue;
  }
#undef GP_CASE
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || parts == 1) return e;
  const int64_t pieces = a.M * ((a.N + 7) / 8);
  hipLaunchKernelGGL((q4_join_kernel<T>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, a,
                     (const float*)a.ws, parts);
  return hipGetLastError();
}

template <class T, int CW, int S, int MT, bool FOUR>
hipError_t rows_launch(const Q4Args& a, int waves, dim3 grid, hipStream_t s) {
  const dim3 block(waves * kWave);
  switch (a.group) {
    case 32: hipLaunchKernelGGL((q4_rows_kernel<T, CW, S, MT, 32, FOUR>), grid, block, 0, s, a); break;
    case 64: hipLaunchKernelGGL((q4_rows_kernel<T, CW, S, MT, 64, FOUR>), grid, block, 0, s, a); break;
    case 128: hipLaunchKernelGGL((q4_rows_kernel<T, CW, S, MT, 128, FOUR>), grid, block, 0, s, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

// Products that run on tiles.  Up to 128 rows small ones do not, up to 64 those
// whose x the kernel for few rows does not read for too many columns, up to 48
// none.  In us, on tiles / by the kernel for few rows:
//    65 and 128 rows: 1,024 columns from 1,024 k   9.6 / 6.6,   9.1 / 6.6
//                     2,048         from 2,048 k  12.1 / 8.4,  11.4 / 8.7
//                     2,048         from 4,096 k  13.8 / 11.6, 15.7 / 11.8  (the rule errs)
//                     1,024         from 16,384 k 20.6 / 30,   20.3 / 32
//                     4,096         from 1,024 k  10.1 / 10.3, 10.3 / 11.4
//                     4,096         from 4,096 k  16.4 / 20.3, 19.3 / 21.5
//   64 rows of 4,096 k: 4,096 columns 16.0 / 12.3, 8,192 19.5 / 14.2, 16,384
//   24.1 / 26.9, 2 x 16,384 35.8 / 53.5; 8,192 from 8,192 24.3 / 23.1
//   48 rows of 4,096 k: 16,384 columns 23.3 / 15.4, 2 x 16,384 35.5 / 29.3
bool on_tiles(int64_t M, int N, int K, int group, int sides) {
  if ((int64_t)((K + group - 1) / group) * N < 4) return false;  // a tile's loads of scales are four wide
  const int64_t n = (int64_t)N * sides;
  return M > 128 || (M > 64 && (n > 2048 || K > 2048)) || (M > 48 && n > 8192);
}

template <class T>
hipError_t launch(const Q4Args& a, int num_cus, hipStream_t s) {
  const int chunks = (a.K + kChunk - 1) / kChunk;
  // One row, and one only: with this kernel and the one for few rows 4,096
  // columns from 4,096 k take 4.4 and 4.8 us, 8,192 from 8,192 7.9 and 8.4, 2 x
  // 16,384 from 4,096 13.5 and 15.2 (the other way round 1,024 from 1,024 3.2 and
  // 3.0, 8,192 from 16,384 17.8 and 14.5); two rows, with digits enough for an
  // fp32 sum, 5.6 and 4.9, 9.2 and 8.2, 14.5 and 15.2, three 6.3 and 4.8.
  if (a.M == 1 && a.N % 2 == 0) {
    int ct = a.N >= 64 * num_cus ? 4 : a.N >= 32 * num_cus ? 2 : 1;
    int kw = 16 / (ct * a.sides);
    while (kw > 1 && kw / 2 >= chunks) kw /= 2;
    const int waves = kw * ct * a.sides;
    const bool z = a.side[0].z || a.side[1].z;
    const TokenLds l = token_lds(a.K, a.group, waves, kw, z);
    if (l.bytes <= kTokenLds) return token_launch<T>(a, waves, ct, kw, l, s);
  }
  if (on_tiles(a.M, a.N, a.K, a.group, a.sides)) {
    TilePlan plan = tile_plan(a.M, a.N, a.K, a.sides, num_cus);
    if (a.ws_bytes < (plan.parts > 1 ? (int64_t)plan.parts * a.sides * a.M * a.N * 4 : 0)) plan.parts = 1;
    return plan.cw == 4   ? tile_launch<T, 4>(a, plan.parts, s)
           : plan.cw == 2 ? tile_launch<T, 2>(a, plan.parts, s)
                          : tile_launch<T, 1>(a, plan.parts, s);
  }
  const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : a.M <= 48 ? 3 : 4;
  // Tiles of 16 columns a wave, both weights' together: as many as leave every
  // CU a workgroup, so that x is read for more columns at once.  (Four with more
  // than 48 rows: a whole chip's products of so many columns run on tiles.)
  const int64_t n = (int64_t)a.N * a.sides;
  int nt = n >= 64 * num_cus && mt < 4 ? 4 : n >= 32 * num_cus ? 2 : 1;
  if ((int64_t)((a.K + a.group - 1) / a.group) * a.N < 4) nt = 1;
  const int cw = nt > a.sides ? nt / a.sides : 1;
  int waves = rows_waves(cw * a.sides, mt);
  while (waves > 2 && waves / 2 >= chunks) waves /= 2;
  const dim3 grid((unsigned)((a.N + 16 * cw - 1) / (16 * cw)), (unsigned)((a.M + 16 * mt - 1) / (16 * mt)));
#define GP_CASE(c, m, four)                                       \
  if (cw == c && a.sides == 1 && mt == m && (a.M <= 4) == four)   \
    return rows_launch<T, c, 1, m, four>(a, waves, grid, s);      \
  if constexpr (c <= 2 && c * m < 8)                              \
    if (cw == c && a.sides == 2 && mt == m && (a.M <= 4) == four) \
      return rows_launch<T, c, 2, m, four>(a, waves, grid, s);
  GP_CASE(1, 1, true) GP_CASE(2, 1, true) GP_CASE(4, 1, true)
  GP_CASE(1, 1, false) GP_CASE(2, 1, false) GP_CASE(4, 1, false)
  GP_CASE(1, 2, false) GP_CASE(2, 2, false) GP_CASE(4, 2, false)
  GP_CASE(1, 3, false) GP_CASE(2, 3, false) GP_CASE(4, 3, false)
  GP_CASE(1, 4, false) GP_CASE(2, 4, false)
#undef GP_CASE
  return hipErrorInvalidValue;
}

}  // namespace

int64_t q4_workspace(int64_t M, int N, int K, int group, int sides, int num_cus) {
  if (!on_tiles(M, N, K, group, sides)) return 0;
  const TilePlan plan = tile_plan(M, N, K, sides, num_cus);
  return plan.parts == 1 ? 0 : (int64_t)plan.parts * sides * M * N * 4;
}

hipError_t q4_launch(const Q4Args& a, int num_cus, hipStream_t s) {
  return a.dtype == GP_DTYPE_BF16 ? launch<BF16>(a, num_cus, s) : launch<F16>(a, num_cus, s);
}

}  // namespace gp
