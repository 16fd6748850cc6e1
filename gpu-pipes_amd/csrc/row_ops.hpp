// What the kernels of a language model's feed-forward half share: loads and
// stores of up to eight 16-bit values, sums over lanes, activations.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/gpipes.h"
#include "gp_device.hpp"
#include "stages.hpp"

namespace gp {

// Eight 16-bit values at an address of any 2-byte alignment: gfx950 takes
// unaligned global accesses, so this is one 16-byte instruction.
typedef unsigned short us8 __attribute__((ext_vector_type(8), aligned(2)));

typedef unsigned short us4 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned short us2 __attribute__((ext_vector_type(2), aligned(2)));

__device__ __forceinline__ u32x4 load16(const half_t* p) { return __builtin_bit_cast(u32x4, *(const us8*)p); }

// The first n of eight 16-bit values, zeros behind them.  BACK: the seven
// values before p may be read (they belong to the same row): the eight that
// end with the n-th are then read in one instruction and moved into place.
template <bool BACK>
__device__ __forceinline__ u32x4 load_raw8(const half_t* p, int n) {
  u32x4 u = {0, 0, 0, 0};
  if (n >= 8) return load16(p);
  if (n <= 0) return u;
  if constexpr (BACK) {
    const u32x4 v = load16(p - (8 - n));
    const int m = 8 - n;  // places too far back
    u32x4 w = m & 4 ? u32x4{v[2], v[3], 0, 0} : v;
    w = m & 2 ? u32x4{w[1], w[2], w[3], 0} : w;
    return m & 1 ? u32x4{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16} : w;
  } else {
    us8 t = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) t[e] = *(const unsigned short*)(p + e);
    return __builtin_bit_cast(u32x4, t);
  }
}

// Eight 16-bit values as fp32.
template <class T>
__device__ __forceinline__ void widen8(u32x4 u, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = T::val(__builtin_bit_cast(half_t, (unsigned short)(u[e] & 0xFFFF)));
    f[2 * e + 1] = T::val(__builtin_bit_cast(half_t, (unsigned short)(u[e] >> 16)));
  }
}

// The first n of eight values as fp32, zeros behind them.
template <class T, bool BACK = false>
__device__ __forceinline__ void load8(const half_t* p, int n, float (&f)[8]) {
  widen8<T>(load_raw8<BACK>(p, n), f);
}

// Stores the first n of eight values, rounded to nearest even.
template <class T>
__device__ __forceinline__ void store8(half_t* p, int n, const float (&f)[8]) {
  u32x4 u;
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = __builtin_bit_cast(unsigned, T::cvt2(f2{f[2 * e], f[2 * e + 1]}));
  if (n >= 8) {
    *(us8*)p = __builtin_bit_cast(us8, u);
  } else if (n > 0) {  // as four, two and one
    if (n & 4) {
      *(us4*)p = __builtin_bit_cast(us4, u32x2{u[0], u[1]});
      p += 4;
      u[0] = u[2], u[1] = u[3];
    }
    if (n & 2) {
      *(us2*)p = __builtin_bit_cast(us2, u[0]);
      p += 2;
      u[0] = u[1];
    }
    if (n & 1) *(unsigned short*)p = (unsigned short)(u[0] & 0xFFFF);
  }
}

// The activations of the stages and SiLU, v / (1 + e^(-v)); at v = -inf, as at
// the others' like, NaN.
__device__ __forceinline__ float apply_act_ext(float v, int act) {
  return act == GP_ACT_SILU ? v * sigmoid(v) : apply_act(v, act);
}

// Eight of them, the choice made once.
__device__ __forceinline__ void apply_act8(float (&v)[8], int act) {
  auto each = [&](auto f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = f(v[e]);
  };
  switch (act) {
    case GP_ACT_RELU: each([](float x) { return relu(x); }); break;
    case GP_ACT_GELU_TANH: each([](float x) { return gelu_tanh(x); }); break;
    case GP_ACT_SIGMOID: each([](float x) { return sigmoid(x); }); break;
    case GP_ACT_SILU: each([](float x) { return x * sigmoid(x); }); break;
    default: break;
  }
}

}  // namespace gp
