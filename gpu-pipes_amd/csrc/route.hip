// Routing of tokens to experts: the k best of E experts for each token and
// their weights, from the router's logits.  No counterpart in the reference.
//
//   s = softmax(l) or sigmoid(l);   c = s + bias, or without a bias the order of l itself
//   the top_groups best of `groups` groups of experts, by their largest c or the sum of their two largest
//   the k best c in those groups, ties to the lowest expert;  w = s, divided by their sum (renorm), times scale
//
// Which of two experts is better can hang on the last bits of their scores, so
// scores that are compared are in 64 bits; without a bias, and with groups by
// their largest, the logits decide and stay in 32.  Weights are made for the
// chosen experts alone, in 64 bits, and rounded once.
//
// A token has 16 lanes up to 256 experts (four tokens a wave, and every exchange
// between lanes a DPP rotation), 64 above.  Bound by instructions: an argument's
// maximum over a token is V compares a lane and four or six exchanges, k times.
#include <hip/hip_runtime.h>

#include "../../include/gpipes.h"
#include "gp_device.hpp"
#include "gp_kernels.hpp"

namespace gp {
namespace {

template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(int, v)));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  const u32x2 u = __builtin_bit_cast(u32x2, v);
  return __builtin_bit_cast(double, u32x2{(unsigned)dpp<CTRL>((int)u[0]), (unsigned)dpp<CTRL>((int)u[1])});
}
// The values that this lane's and its partner's half (16 or 32 lanes away) hold.
template <int HALF>
__device__ __forceinline__ void halves(unsigned v, unsigned& a, unsigned& b) {
  if constexpr (HALF == 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    a = p[0], b = p[1];
  } else {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    a = p[0], b = p[1];
  }
}
template <int HALF>
__device__ __forceinline__ void halves(int v, int& a, int& b) {
  unsigned x, y;
  halves<HALF>((unsigned)v, x, y);
  a = (int)x, b = (int)y;
}
template <int HALF>
__device__ __forceinline__ void halves(float v, float& a, float& b) {
  unsigned x, y;
  halves<HALF>(__builtin_bit_cast(unsigned, v), x, y);
  a = __builtin_bit_cast(float, x), b = __builtin_bit_cast(float, y);
}
template <int HALF>
__device__ __forceinline__ void halves(double v, double& a, double& b) {
  const u32x2 u = __builtin_bit_cast(u32x2, v);
  unsigned x0, y0, x1, y1;
  halves<HALF>(u[0], x0, y0), halves<HALF>(u[1], x1, y1);
  a = __builtin_bit_cast(double, u32x2{x0, x1}), b = __builtin_bit_cast(double, u32x2{y0, y1});
}

// f over the values of a token's lanes, the same in each of them (f commutes).
template <int LPT, class V, class F>
__device__ __forceinline__ V over_token(V v, F f) {
  v = f(v, dpp<0x128>(v));  // row_ror:8, 4, 2, 1
  v = f(v, dpp<0x124>(v));
  v = f(v, dpp<0x122>(v));
  v = f(v, dpp<0x121>(v));
  if constexpr (LPT == 64) {
    V a, b;
    halves<16>(v, a, b), v = f(a, b);
    halves<32>(v, a, b), v = f(a, b);
  }
  return v;
}
// The best (key, index) over a token's lanes: the largest key, of equal ones the lowest index.
template <int LPT, class K>
__device__ __forceinline__ void best_of_token(K& k, int& i) {
  auto take = [&](K k2, int i2) {
    const bool b = k2 > k || (k2 == k && i2 < i);
    k = b ? k2 : k, i = b ? i2 : i;
  };
  take(dpp<0x128>(k), dpp<0x128>(i));
  take(dpp<0x124>(k), dpp<0x124>(i));
  take(dpp<0x122>(k), dpp<0x122>(i));
  take(dpp<0x121>(k), dpp<0x121>(i));
  if constexpr (LPT == 64) {
    K ka, kb;
    int ia, ib;
    halves<16>(k, ka, kb), halves<16>(i, ia, ib), k = ka, i = ia, take(kb, ib);
    halves<32>(k, ka, kb), halves<32>(i, ia, ib), k = ka, i = ia, take(kb, ib);
  }
}

__device__ __forceinline__ float logit(const void* l, int64_t at, int dtype) {
  if (dtype == GP_DTYPE_F32) return ((const float*)l)[at];
  const half_t h = ((const half_t*)l)[at];
  return dtype == GP_DTYPE_F16 ? F16::val(h) : BF16::val(h);
}
__device__ __forceinline__ double sigmoid64(float l) { return 1.0 / (1.0 + exp(-(double)l)); }

constexpr int kWaves = 4;

// Lane i of a token holds experts i, i + LPT, ...  K: the keys' type, double where scores are compared.
template <class K, int LPT, int V>
__global__ __launch_bounds__(64 * kWaves) void route_experts_kernel(RouteExpertsArgs p) {
  constexpr int TPW = 64 / LPT, VG = kRouteMaxGroups / LPT, VK = (kRouteMaxK + LPT - 1) / LPT;
  constexpr bool D = sizeof(K) == 8;
  extern __shared__ __attribute__((aligned(16))) char mem[];  // of a wave: a token's keys one after the other
  const K none = -(K)__builtin_inff();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & (LPT - 1);
  const int64_t token = ((int64_t)blockIdx.x * kWaves + wave) * TPW + lane / LPT;
  const int64_t t = token < p.T ? token : p.T - 1;  // every lane takes part in the exchanges
  const int E = p.E;
  const float inf = __builtin_inff();

  float l[V];
  float top = -inf;
  bool bad = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * LPT + i;
    l[v] = e < E ? logit(p.logits, t * E + e, p.dtype) : -inf;
    bad |= l[v] != l[v];
    top = l[v] > top ? l[v] : top;
  }
  top = over_token<LPT>(top, [](float a, float b) { return a > b ? a : b; });
  const bool softmax = p.score == GP_SCORE_SOFTMAX;
  bad |= softmax && top == inf;

  // The softmax's denominator, where scores themselves are asked for.
  double sum = 1.0;
  if (softmax && (D || !p.renorm)) {
    sum = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += l[v] == -inf ? 0.0 : exp((double)l[v] - (double)top);
    sum = over_token<LPT>(sum, [](double a, double b) { return a + b; });
  }
  auto score = [&](float x) { return softmax ? exp((double)x - (double)top) / sum : sigmoid64(x); };

  K key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    key[v] = (K)l[v];
    if constexpr (D) {
      if (p.bias && l[v] != -inf) {
        key[v] = score(l[v]) + (double)p.bias[v * LPT + i];
        bad |= key[v] != key[v];
      }
    }
  }

  if (p.top_groups < p.groups) {
    K* const rank = (K*)mem + (wave * TPW + lane / LPT) * E;
    const int size = E / p.groups;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = v * LPT + i;
      K r = key[v];
      if constexpr (D)
        if (!p.bias && l[v] != -inf) r = score(l[v]);
      if (e < E) rank[e] = r;
    }
    lds_barrier();
    K g[VG];
    unsigned long long kept = 0;
#pragma unroll
    for (int v = 0; v < VG; ++v) {
      const int gi = v * LPT + i;
      K a = none, b = none;  // the group's two best
      if (gi < p.groups)
        for (int e = 0; e < size; ++e) {
          const K r = rank[gi * size + e];
          b = r > a ? a : r > b ? r : b;
          a = r > a ? r : a;
        }
      g[v] = p.group_score == GP_GROUP_TOP2 && b > none ? a + b : a;
    }
    for (int n = 0; n < p.top_groups; ++n) {
      K bk = none;
      int bi = 1 << 20;
#pragma unroll
      for (int v = 0; v < VG; ++v)
        if (g[v] > bk) bk = g[v], bi = v * LPT + i;
      best_of_token<LPT>(bk, bi);
      if (bk > none) kept |= 1ull << bi;  // of groups with no expert left none is kept
#pragma unroll
      for (int v = 0; v < VG; ++v)
        if (bi == v * LPT + i) g[v] = none;
    }
    const float per = 1.f / (float)size;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int of = (int)(((float)(v * LPT + i) + 0.5f) * per);  // exact: below 2^10
      if (!(kept >> (of & 63) & 1)) key[v] = none;
    }
  }

  // One after the other; lane n % LPT keeps the n-th.
  int id[VK];
#pragma unroll
  for (int s = 0; s < VK; ++s) id[s] = -1;
  for (int n = 0; n < p.k; ++n) {
    K bk = none;
    int bi = 1 << 20;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v] > bk) bk = key[v], bi = v * LPT + i;
    best_of_token<LPT>(bk, bi);
    if (!(bk > none)) bi = -1;
#pragma unroll
    for (int s = 0; s < VK; ++s)
      if (n == s * LPT + i) id[s] = bi;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (bi == v * LPT + i) key[v] = none;
  }

  // Weights: of a softmax that is divided by the chosen ones' sum, relative to the largest of them.
  const bool relative = softmax && p.renorm;
  float x[VK], xtop = -inf;
#pragma unroll
  for (int s = 0; s < VK; ++s) {
    x[s] = id[s] < 0 ? -inf : logit(p.logits, t * E + id[s], p.dtype);
    xtop = x[s] > xtop ? x[s] : xtop;
  }
  if (relative) xtop = over_token<LPT>(xtop, [](float a, float b) { return a > b ? a : b; });
  double w[VK], total = 0.0;
#pragma unroll
  for (int s = 0; s < VK; ++s) {
    w[s] = id[s] < 0 ? 0.0 : relative ? exp((double)x[s] - (double)xtop) : score(x[s]);
    total += w[s];
  }
  if (p.renorm) total = over_token<LPT>(total, [](double a, double b) { return a + b; });
  const int any = over_token<LPT>((int)bad, [](int a, int b) { return a | b; });
#pragma unroll
  for (int s = 0; s < VK; ++s) {
    const int n = s * LPT + i;
    if (n >= p.k || token >= p.T) continue;
    const double v = p.renorm ? (total > 0.0 ? w[s] / total : 0.0) : w[s];
    p.weights[t * p.k + n] = any ? __builtin_nanf("") : (float)(v * (double)p.scale);
    p.ids[t * p.k + n] = any ? n : id[s];
  }
}

template <class K, int LPT, int V>
hipError_t launch_one(const RouteExpertsArgs& a, hipStream_t s) {
  const int64_t per = kWaves * (64 / LPT);
  const int bytes = a.top_groups < a.groups ? (int)(per * a.E * sizeof(K)) : 0;
  const auto kern = &route_experts_kernel<K, LPT, V>;
  hipLaunchKernelGGL(kern, dim3((unsigned)((a.T + per - 1) / per)), dim3(64 * kWaves), bytes, s, a);
  return hipGetLastError();
}

template <class K>
hipError_t launch(const RouteExpertsArgs& a, hipStream_t s) {
  if (a.E <= 16) return launch_one<K, 16, 1>(a, s);
  if (a.E <= 32) return launch_one<K, 16, 2>(a, s);
  if (a.E <= 64) return launch_one<K, 16, 4>(a, s);
  if (a.E <= 128) return launch_one<K, 16, 8>(a, s);
  if (a.E <= 256) return launch_one<K, 16, 16>(a, s);
  if (a.E <= 512) return launch_one<K, 64, 8>(a, s);
  return launch_one<K, 64, 16>(a, s);
}

}  // namespace

hipError_t route_experts_launch(const RouteExpertsArgs& a, hipStream_t s) {
  const bool scores = a.bias || (a.top_groups < a.groups && a.group_score == GP_GROUP_TOP2);
  return scores ? launch<double>(a, s) : launch<float>(a, s);
}

}  // namespace gp
