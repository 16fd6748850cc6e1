// Routing of tokens to experts: the k best of E experts for each token and
// their weights, from the router's logits.  No counterpart in the reference.
//
//   s = softmax(l) or sigmoid(l);   c = s + bias, or without a bias the order of l itself
//   the top_groups best of `groups` groups of experts, by their largest c or the sum of their two largest
//   the k best c in those groups, ties to the lowest expert;  w = s, divided by their sum (renorm), times scale
//
// Which of two experts is better can hang on the last bits of their scores, so
// the order is that of scores in 64 bits: scores in 32 bits decide where they are
// further apart than they can be off, and a wave with a token whose choice is
// closer than that makes its choices again in 64.  Without a bias, and with groups
// by their largest, the logits decide.  Weights are made for the chosen experts
// alone, in 64 bits, and rounded once.
//
// How far scores in 32 bits can be off, in units u = 2^-24: an exponential by 2 of
// itself (v_exp_f32) and its argument's roundings, a reciprocal by 2 (v_rcp_f32).
// Sigmoid, s = 1 / (1 + e): 0.23 (argument; s (1 - s) |l| < 0.23) + 0.5 (exponential;
// s (1 - s) <= 1/4) + 3 (sum, reciprocal), and c's own rounding |c|: below 2^-21 of |c|
// or of 1, whichever is more.  Softmax: 1 + 2 + 3 for e and the reciprocal, and
// its sum, of up to 22 additions and of exponentials whose arguments are 8 on
// average at most, by 22 + 2 * 8 + 2 of itself: below 2^-18.
//
// A token has 16 lanes up to 256 experts (four tokens a wave, and every exchange
// between lanes a DPP rotation), 64 above.  Bound by instructions: an argument's
// maximum over a token is V compares a lane and four or six exchanges, k times.
// 16,384 tokens to 6 of 128 experts in 8 groups: 11.8 us among other calls, 11.9 in a
// graph, 1,119 vector instructions a wave (814 without groups); with all scores in
// 64 bits 16.6 in a graph.
#include <hip/hip_runtime.h>

#include <type_traits>

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
__device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)dpp<CTRL>((int)v);
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
__device__ __forceinline__ float logit(const void* l, int64_t at, int dtype) {
  if (dtype == GP_DTYPE_F32) return ((const float*)l)[at];
  const half_t h = ((const half_t*)l)[at];
  return dtype == GP_DTYPE_F16 ? F16::val(h) : BF16::val(h);
}
__device__ __forceinline__ double sigmoid64(float l) { return 1.0 / (1.0 + exp(-(double)l)); }

constexpr int kWaves = 4;
constexpr int kRouteLds = 128 + 136;  // bytes a token: sixteen keys of 64 bits, kRouteMaxK + 1 experts (and a gap)

// What a token's lanes know of it: lane i holds experts i, i + LPT, ...  No
// logit is NaN, and none makes its c one: a row that has such has -inf here.
template <int V>
struct Token {
  float l[V];  // logits, -inf behind the last expert
  float top;   // the largest
  int64_t t;   // the token
  float bias[V];
};

// A wave's own LDS: what its lanes have written is there for all of them.
__device__ __forceinline__ void wave_lds() {
  compiler_fence();
  __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
  compiler_fence();
}

// The largest of the keys and the lowest expert that has it; it is taken out of
// them.  No key is NaN: lanes would come to different largest ones, and to no expert.
template <int LPT, class K, int V>
__device__ __forceinline__ int take_best(K (&key)[V], int i, K& best) {
  K m = key[0];
#pragma unroll
  for (int v = 1; v < V; ++v) m = key[v] > m ? key[v] : m;
  best = over_token<LPT>(m, [](K a, K b) { return a > b ? a : b; });
  int at = 1 << 20;
#pragma unroll
  for (int v = V - 1; v >= 0; --v) at = key[v] == best ? v * LPT + i : at;
  at = over_token<LPT>(at, [](int a, int b) { return a < b ? a : b; });
#pragma unroll
  for (int v = 0; v < V; ++v) key[v] = at == v * LPT + i ? -(K)__builtin_inff() : key[v];
  return at;
}

// Keys of a token's experts: the logits, or (SCORES) c in K's precision, -inf for
// those that cannot be chosen.
template <class K, bool SCORES, int LPT, int V>
__device__ __forceinline__ void make_keys(const RouteExpertsArgs& p, const Token<V>& x, K (&key)[V], K (&rank)[V]) {
  const bool softmax = p.score == GP_SCORE_SOFTMAX;
  const float inf = __builtin_inff();
  K sum = 1;
  if (SCORES && softmax) {
    sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if constexpr (sizeof(K) == 8)
        sum += x.l[v] == -inf ? 0.0 : exp((double)x.l[v] - (double)x.top);
      else
        sum += x.l[v] == -inf ? 0.f : __builtin_amdgcn_exp2f((x.l[v] - x.top) * 1.4426950408889634f);
    }
    sum = over_token<LPT>(sum, [](K a, K b) { return a + b; });
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    key[v] = rank[v] = (K)x.l[v];
    if constexpr (SCORES) {
      K s;
      if constexpr (sizeof(K) == 8) {
        s = softmax ? exp((double)x.l[v] - (double)x.top) / sum : sigmoid64(x.l[v]);
      } else {
        const float e = __builtin_amdgcn_exp2f((softmax ? x.l[v] - x.top : -x.l[v]) * 1.4426950408889634f);
        s = softmax ? e * __builtin_amdgcn_rcpf((float)sum) : __builtin_amdgcn_rcpf(1.f + e);
      }
      const bool out = x.l[v] == -inf;
      if (p.bias) {
        key[v] = rank[v] = out ? key[v] : s + (K)x.bias[v];
      } else {
        rank[v] = out ? key[v] : s;
      }
    }
  }
}

// Leaves the keys of the top_groups best groups.  at: the token's place in the
// wave's LDS.  off: how far a c can be from its value, of itself or of 1 (0: not at
// all).  Whether every group that is kept is certain to be better than every
// other one comes back.  A group's sum is as far from its value as its terms are,
// however small it is itself: terms of |c| <= m and the sum's rounding 2.25 off m,
// the bound's own 0.25 off m, so 3 off m.  A sum of finite terms above fp32's range is
// no value at all; for one below it (a group masked by the type's lowest value)
// stands the lowest value, with -inf as its least: 16,384 tokens with such a group
// 12.9 us instead of 20.7 in 64 bits.  A sum with an infinite term is exact.
template <class K, int LPT, int V>
__device__ __forceinline__ bool keep_groups(const RouteExpertsArgs& p, K (&key)[V], const K (&rank)[V], int i, K* at, float off) {
  const K none = -(K)__builtin_inff();
  const int size = p.E / p.groups;
  wave_lds();  // what was there is done with
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (v * LPT + i < p.E) at[v * LPT + i] = rank[v];
  wave_lds();
  bool sure = true;
  unsigned long long kept = 0;
  auto select = [&](auto vg) {
    constexpr int VG = decltype(vg)::value;
    K g[VG];
    float least[VG], most[VG];  // what the group's value may be
    bool lost = false;          // a sum above fp32's range
#pragma unroll
    for (int v = 0; v < VG; ++v) {
      const int gi = v * LPT + i < p.groups ? v * LPT + i : p.groups - 1;
      K a = none, b = none;  // the group's two best
      for (int e = 0; e < size; ++e) {
        const K r = at[gi * size + e];
        if constexpr (sizeof(K) == 4) {
          b = __builtin_amdgcn_fmed3f(a, b, r);
          a = fmaxf(a, r);
        } else {
          const K low = r > a ? a : r;
          b = low > b ? low : b;
          a = r > a ? r : a;
        }
      }
      const bool two = p.group_score == GP_GROUP_TOP2 && b > none;
      g[v] = two ? a + b : a;
      if constexpr (sizeof(K) == 4) {
        // an infinite m makes NaNs here, which the minimum and the maximum below pass over
        const float d = 3.f * off * fmaxf(fmaxf(fabsf(a), two ? fabsf(b) : 1.f), 1.f);
        lost |= two && a < -none && g[v] == -none;
        g[v] = two ? fmaxf(g[v], -3.4028234664e38f) : g[v];
        least[v] = g[v] - d;  // below the lowest value: -inf, d being more than half its step there
        most[v] = v * LPT + i < p.groups ? g[v] + d : none;
      }
      g[v] = v * LPT + i < p.groups ? g[v] : none;
    }
    for (int n = 0; n < p.top_groups; ++n) {
      K best;
      const int of = take_best<LPT>(g, i, best);
      if (best > none) kept |= 1ull << (of & 63);  // of groups with no expert left none is kept
    }
    if constexpr (sizeof(K) == 4) {
      if (off > 0.f) {
        float in = -none, out = lost ? -none : none;
#pragma unroll
        for (int v = 0; v < VG; ++v) {
          const bool is = kept >> (v * LPT + i & 63) & 1;
          in = fminf(in, is ? least[v] : -none);
          out = fmaxf(out, is ? none : most[v]);
        }
        in = over_token<LPT>(in, [](float a, float b) { return fminf(a, b); });
        out = over_token<LPT>(out, [](float a, float b) { return fmaxf(a, b); });
        sure = in > out;
      }
    }
  };
  if (p.groups <= LPT)
    select(std::integral_constant<int, 1>{});
  else
    select(std::integral_constant<int, kRouteMaxGroups / LPT>{});
  const float per = 1.f / (float)size;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int of = (int)(((float)(v * LPT + i) + 0.5f) * per);  // exact: below 2^10
    if (!(kept >> (of & 63) & 1)) key[v] = none;
  }
  return sure;
}

// A token's experts in the definition's order, lane n % LPT keeping the n-th in
// id[n / LPT]: scores (K double) in 64 bits, logits (float) as they are.
template <class K, bool SCORES, int LPT, int V, int VK>
__device__ __forceinline__ void choose(const RouteExpertsArgs& p, const Token<V>& x, int i, K* at, int (&id)[VK]) {
  K key[V], rank[V];
  make_keys<K, SCORES, LPT>(p, x, key, rank);
  if (p.top_groups < p.groups) keep_groups<K, LPT>(p, key, rank, i, at, 0.f);
#pragma unroll
  for (int s = 0; s < VK; ++s) id[s] = -1;
  for (int n = 0; n < p.k; ++n) {
    K best;
    const int e = take_best<LPT>(key, i, best);
#pragma unroll
    for (int s = 0; s < VK; ++s)
      if (n == s * LPT + i && best > -(K)__builtin_inff()) id[s] = e;
  }
}

// The same in fewer instructions, with keys of 32 bits of which the best one is a
// minimum: the distance d from the largest key, less its last bits, and in their
// place which of its lane's experts it is.  16-bit logits fit as they are, with the
// expert below them (of equal ones the lowest comes first), and no choice is in
// doubt.  Else one is where the next d is no further than scores, or what d has
// lost, may be off: then the k best and those after them that are too close to the
// last, up to sixteen, are put in order by their keys in 64 bits, one a lane.  What
// that does not settle (a softmax, whose sum is needed in 64 bits, groups too close
// to each other, more candidates) comes back as false.  list, cand: a token's places
// in LDS for its experts and sixteen keys.
template <bool SCORES, int LPT, int V>
__device__ __forceinline__ bool choose_fast(const RouteExpertsArgs& p, const Token<V>& x, int i, float* at, int* list, double* cand) {
  constexpr unsigned mask = V <= 1 ? 0 : V <= 2 ? 1 : V <= 4 ? 3 : V <= 8 ? 7 : 15;
  constexpr float lost = 2.f * (float)(mask + 1) / (1 << 23);  // of d: its last bits, and two roundings
  const float inf = __builtin_inff();
  const float off = !SCORES ? 0.f : p.score == GP_SCORE_SOFTMAX ? 1.f / (1 << 18) : 1.f / (1 << 21);
  const bool exact = !SCORES && p.dtype != GP_DTYPE_F32;
  float key[V], rank[V];
  make_keys<float, SCORES, LPT>(p, x, key, rank);
  bool sure = true;
  if (p.top_groups < p.groups) sure = keep_groups<float, LPT>(p, key, rank, i, at, off);
  float top = -inf;
#pragma unroll
  for (int v = 0; v < V; ++v) top = fmaxf(top, key[v]);
  top = over_token<LPT>(top, [](float a, float b) { return fmaxf(a, b); });
  sure &= exact || top < inf;
  unsigned u[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    unsigned k;
    if (exact) {
      // a 16-bit logit's bits are the upper ones of bf16's float; fp16 goes back to its own
      const float l = key[v] + 0.f;  // -0 is 0
      const unsigned h = p.dtype == GP_DTYPE_BF16 ? __builtin_bit_cast(unsigned, l) >> 16
                                                  : (unsigned)__builtin_bit_cast(unsigned short, (half_t)l);
      k = ((h & 0x8000u ? h : ~h & 0x7FFFu) << 16) | (unsigned)(v * LPT + i);  // larger ones first
    } else {
      k = (__builtin_bit_cast(unsigned, top - key[v]) & ~mask) | v;
    }
    u[v] = key[v] == -inf ? ~0u : k;
  }
  float last = 0.f;
  unsigned m;
  bool found, close = false;  // too close to the one before
  // The n-th best: out of the keys, and its expert at list[n].
  auto next = [&](int n) {
    unsigned mine = u[0];
#pragma unroll
    for (int v = 1; v < V; ++v) mine = u[v] < mine ? u[v] : mine;
    m = over_token<LPT>(mine, [](unsigned a, unsigned b) { return a < b ? a : b; });
#pragma unroll
    for (int v = 0; v < V; ++v) u[v] = u[v] == m ? ~0u : u[v];
    found = m != ~0u;
    if (mine == m) list[n] = !found ? -1 : exact ? (int)(m & 0xFFFFu) : (int)(m & mask) * LPT + i;
    if (!exact) {
      const float d = __builtin_bit_cast(float, m & ~mask);
      close = found && !(d - last > 2.f * off * fmaxf(fmaxf(fabsf(top), fabsf(top - d)), 1.f) + lost * d);
      last = d;
      // two lanes with one key: both were taken out
      const unsigned long long won = __ballot(mine == m) >> (threadIdx.x & 63 & ~(LPT - 1));
      sure &= !found || __popcll(LPT == 64 ? won : won & 0xFFFF) == 1;
    }
  };
  bool doubt = false;
  for (int n = 0; n < p.k + !exact; ++n) {
    next(n);
    doubt |= n > 0 && close;
  }
  if (exact || !__any(doubt)) return sure;
  constexpr int MOST = 16;
  if ((SCORES && p.score == GP_SCORE_SOFTMAX) || p.k >= MOST) return sure && !doubt;
  // candidates: k, and while each is too close to the one before, the next ones
  int q = p.k;
  bool open = close;
  for (int n = p.k; __any(open); ++n) {
    if (n >= MOST) {
      sure &= !open;
      break;
    }
    if (n > p.k) {
      next(n);
      open &= close;
    }
    q += open;
  }
  wave_lds();
  const bool one = i < q && i < MOST;
  int e = one ? list[i] : -1;
  double c = -(double)inf;
  if ((unsigned)e < (unsigned)p.E) {
    const float l = logit(p.logits, x.t * p.E + e, p.dtype);
    c = SCORES && p.bias ? sigmoid64(l) + (double)p.bias[e] : (double)l;
  }
  if (i < MOST) cand[i] = c;
  wave_lds();
  int better = 0;
#pragma unroll 1
  for (int n = 0; n < MOST; ++n) {
    const double o = cand[n];
    const int oe = n < q ? list[n] : -1;
    better += oe >= 0 && (o > c || (o == c && oe < e));
  }
  wave_lds();
  if (e >= 0 && better < p.k) list[better] = e;
  return sure;
}

template <bool SCORES, int LPT, int V>
__global__ __launch_bounds__(64 * kWaves) void route_experts_kernel(RouteExpertsArgs p) {
  constexpr int TPW = 64 / LPT, VK = (kRouteMaxK + LPT - 1) / LPT;
  extern __shared__ __attribute__((aligned(16))) char mem[];  // each token's choice, then (with groups) its keys
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & (LPT - 1);
  const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t token = (block * kWaves + wave) * TPW + lane / LPT;
  const int64_t t = token < p.T ? token : p.T - 1;  // every lane takes part in the exchanges
  const float inf = __builtin_inff();
  const bool softmax = p.score == GP_SCORE_SOFTMAX;

  // loads under a condition each would be waited for one by one: the last expert's again instead
  Token<V> x;
  x.t = t;
  if (p.dtype == GP_DTYPE_F32) {
#pragma unroll
    for (int v = 0; v < V; ++v) x.l[v] = ((const float*)p.logits)[t * p.E + (v * LPT + i < p.E ? v * LPT + i : p.E - 1)];
  } else {
    half_t h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = ((const half_t*)p.logits)[t * p.E + (v * LPT + i < p.E ? v * LPT + i : p.E - 1)];
#pragma unroll
    for (int v = 0; v < V; ++v) x.l[v] = p.dtype == GP_DTYPE_F16 ? F16::val(h[v]) : BF16::val(h[v]);
  }
  if (SCORES && p.bias) {
#pragma unroll
    for (int v = 0; v < V; ++v) x.bias[v] = p.bias[v * LPT + i < p.E ? v * LPT + i : p.E - 1];
  }
  // A row with a NaN (scores are 0 to 1, so c is one where the logit or the bias is) or, with softmax, a +inf
  // has no choice to make: to what follows its experts are as those that cannot be chosen.
  x.top = -inf;
  bool nan = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    x.l[v] = v * LPT + i < p.E ? x.l[v] : -inf;
    nan |= x.l[v] != x.l[v];
    if (SCORES && p.bias) nan |= x.bias[v] != x.bias[v] && x.l[v] > -inf;
    x.top = x.l[v] > x.top ? x.l[v] : x.top;
  }
  x.top = over_token<LPT>(x.top, [](float a, float b) { return a > b ? a : b; });
  nan |= softmax && x.top == inf;
  const bool bad = over_token<LPT>((int)nan, [](int a, int b) { return a | b; });
  x.top = bad ? -inf : x.top;
#pragma unroll
  for (int v = 0; v < V; ++v) x.l[v] = bad ? -inf : x.l[v];

  // 32 bits settle nearly every token; where a choice is too close for them, the wave makes its choices again.
  int id[VK];
  typedef typename std::conditional<SCORES, double, float>::type K;
  const int place = wave * TPW + lane / LPT;
  double* const cand = (double*)mem + place * 16;
  int* const list = (int*)(mem + kWaves * TPW * 128) + place * (kRouteMaxK + 1);
  K* const at = (K*)(mem + kRouteLds * kWaves * TPW) + place * p.E;
  const bool sure = choose_fast<SCORES, LPT, V>(p, x, i, (float*)at, list, cand);
  wave_lds();
#pragma unroll
  for (int s = 0; s < VK; ++s) id[s] = s * LPT + i < p.k ? list[s * LPT + i] : -1;
  if (__any(!sure)) choose<K, SCORES, LPT, V>(p, x, i, at, id);

  // Weights: of a softmax that is divided by the chosen ones' sum, relative to the largest of them.
  const bool relative = softmax && p.renorm;
  double sum = 1.0;
  if (softmax && !p.renorm) {
    sum = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += x.l[v] == -inf ? 0.0 : exp((double)x.l[v] - (double)x.top);
    sum = over_token<LPT>(sum, [](double a, double b) { return a + b; });
  }
  float l[VK], ltop = -inf;
#pragma unroll
  for (int s = 0; s < VK; ++s) {
    l[s] = -inf;
    if (s * LPT < p.k && (unsigned)id[s] < (unsigned)p.E) l[s] = logit(p.logits, t * p.E + id[s], p.dtype);
    ltop = l[s] > ltop ? l[s] : ltop;
  }
  if (relative) ltop = over_token<LPT>(ltop, [](float a, float b) { return a > b ? a : b; });
  double w[VK], total = 0.0;
#pragma unroll
  for (int s = 0; s < VK; ++s) {
    w[s] = 0.0;
    if (s * LPT < p.k && id[s] >= 0) {
      w[s] = softmax ? exp((double)l[s] - (double)(relative ? ltop : x.top)) : sigmoid64(l[s]);
      if (!relative) w[s] /= sum;
    }
    total += w[s];
  }
  if (p.renorm) total = over_token<LPT>(total, [](double a, double b) { return a + b; });
#pragma unroll
  for (int s = 0; s < VK; ++s) {
    const int n = s * LPT + i;
    if (n >= p.k || token >= p.T) continue;
    const double v = !p.renorm ? w[s] : total > 0.0 ? w[s] / total : 0.0;
    p.weights[t * p.k + n] = bad ? __builtin_nanf("") : (float)(v * (double)p.scale);
    p.ids[t * p.k + n] = bad ? n : id[s];
  }
}

template <bool SCORES, int LPT, int V>
hipError_t launch_one(const RouteExpertsArgs& a, hipStream_t s) {
  const int64_t per = kWaves * (64 / LPT);
  const int bytes = (int)per * (kRouteLds + (a.top_groups < a.groups ? a.E * (SCORES ? 8 : 4) : 0));
  const auto kern = &route_experts_kernel<SCORES, LPT, V>;
  // a launch holds fewer than 2^32 threads along an axis
  const int64_t n = (a.T + per - 1) / per, most = 1 << 20, y = (n + most - 1) / most;
  hipLaunchKernelGGL(kern, dim3((unsigned)((n + y - 1) / y), (unsigned)y), dim3(64 * kWaves), bytes, s, a);
  return hipGetLastError();
}

template <bool SCORES>
hipError_t launch(const RouteExpertsArgs& a, hipStream_t s) {
  if (a.E <= 16) return launch_one<SCORES, 16, 1>(a, s);
  if (a.E <= 32) return launch_one<SCORES, 16, 2>(a, s);
  if (a.E <= 64) return launch_one<SCORES, 16, 4>(a, s);
  if (a.E <= 128) return launch_one<SCORES, 16, 8>(a, s);
  if (a.E <= 256) return launch_one<SCORES, 16, 16>(a, s);
  if (a.E <= 512) return launch_one<SCORES, 64, 8>(a, s);
  return launch_one<SCORES, 64, 16>(a, s);
}

}  // namespace

hipError_t route_experts_launch(const RouteExpertsArgs& a, hipStream_t s) {
  const bool scores = a.bias || (a.top_groups < a.groups && a.group_score == GP_GROUP_TOP2);
  return scores ? launch<true>(a, s) : launch<false>(a, s);
}

}  // namespace gp
