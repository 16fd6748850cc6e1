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

// The first n of eight values as fp32, zeros behind them.
template <class T>
__device__ __forceinline__ void load8(const half_t* p, int n, float (&f)[8]) {
  us8 u = {0, 0, 0, 0, 0, 0, 0, 0};
  if (n >= 8) {
    u = *(const us8*)p;
  } else if (n > 0) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) u[e] = *(const unsigned short*)(p + e);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = T::val(__builtin_bit_cast(half_t, (unsigned short)u[e]));
}

// Stores the first n of eight values, rounded to nearest even.
template <class T>
__device__ __forceinline__ void store8(half_t* p, int n, const float (&f)[8]) {
  us8 u;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const h2 r = T::cvt2(f2{f[e], f[e + 1]});
    u[e] = __builtin_bit_cast(unsigned short, (half_t)r[0]);
    u[e + 1] = __builtin_bit_cast(unsigned short, (half_t)r[1]);
  }
  if (n >= 8) {
    *(us8*)p = u;
  } else if (n > 0) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) *(unsigned short*)(p + e) = u[e];
  }
}

// The activations of the stages and SiLU, v / (1 + e^(-v)); at v = -inf, as at
// the others' like, NaN.
__device__ __forceinline__ float apply_act_ext(float v, int act) {
  return act == GP_ACT_SILU ? v * sigmoid(v) : apply_act(v, act);
}

}  // namespace gp
