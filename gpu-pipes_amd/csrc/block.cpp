// C ABI of the operators around a language model's feed-forward half: the norms
// with the residual (gp_residual_norm_out), the products with 4-bit weights
// (gp_q4_gemm_out, gp_q4_gated_out), those in 8-bit integers (gp_i8_gemm_out,
// gp_i8_gated_out), the routing to experts (gp_route_out) and their feed-forward
// block (gp_i8_experts_out).  Argument checks
// and dispatch; the kernels are in residual_norm.hip, q4.hip, i8.hip and route.hip.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/gpipes.h"
#include "gp_host.hpp"
#include "gp_kernels.hpp"

namespace gp {
namespace {

int check_dtype(int dtype) {
  if (dtype != GP_DTYPE_F16 && dtype != GP_DTYPE_BF16) return fail(GP_ERR_INVALID_ARG, "unknown dtype %d", dtype);
  return GP_OK;
}

int check_rows(int64_t M) {
  if (M < 0) return fail(GP_ERR_INVALID_ARG, "M must be >= 0 (got %lld)", (long long)M);
  if (M > (int64_t(1) << 40)) return fail(GP_ERR_SHAPE, "M too large (%lld)", (long long)M);
  return GP_OK;
}

int check_act_ext(int act) {
  if (act < GP_ACT_NONE || act > GP_ACT_SILU) return fail(GP_ERR_INVALID_ARG, "unknown activation %d", act);
  return GP_OK;
}

int check_norm(int kind, const void* gamma, const void* beta, float eps, const char* name) {
  if (kind != GP_NORM_NONE && kind != GP_NORM_LAYER && kind != GP_NORM_RMS)
    return fail(GP_ERR_INVALID_ARG, "unknown %s norm %d", name, kind);
  if (kind == GP_NORM_NONE) {
    if (gamma || beta) return fail(GP_ERR_INVALID_ARG, "%s norm is none: its gamma and beta must be NULL", name);
  } else if (!(eps >= 0.f) || std::isinf(eps)) {
    return fail(GP_ERR_INVALID_ARG, "the %s norm's eps must be >= 0 and finite", name);
  }
  return GP_OK;
}

// Whether `n` values of 16 bits at a and `m` at b have memory in common (NULL has none).
bool meet(const void* a, int64_t n, const void* b, int64_t m) {
  return a && b && (uintptr_t)a < (uintptr_t)b + 2 * (uintptr_t)m && (uintptr_t)b < (uintptr_t)a + 2 * (uintptr_t)n;
}

constexpr int64_t kQ4MaxDim = int64_t(1) << 20;

int check16(const void* p, const char* name, bool needed) {
  if (!p) return needed ? fail(GP_ERR_INVALID_ARG, "%s is NULL", name) : GP_OK;
  if (!aligned16(p)) return fail(GP_ERR_ALIGN, "%s must be 16-byte aligned", name);
  return GP_OK;
}

int q4_check_shape(int64_t M, int64_t N, int64_t K, int group) {
  const int rc = check_rows(M);
  if (rc) return rc;
  if (group != 32 && group != 64 && group != 128)
    return fail(GP_ERR_SHAPE, "group must be 32, 64 or 128 (got %d)", group);
  if (K < 8 || K % 8 || K > 65536) return fail(GP_ERR_SHAPE, "K must be a multiple of 8 in [8, 65536] (got %lld)", (long long)K);
  if (N < 1 || N > kQ4MaxDim) return fail(GP_ERR_SHAPE, "N must be in [1, %lld] (got %lld)", (long long)kQ4MaxDim, (long long)N);
  if (K * N / 2 >= (int64_t(1) << 31)) return fail(GP_ERR_SHAPE, "a weight must be smaller than 2 GiB");
  if (M > (int64_t(1) << 21)) return fail(GP_ERR_SHAPE, "M must be at most 2097152 (got %lld)", (long long)M);
  return GP_OK;
}

int q4_run(const Q4Args& a, int64_t N, int64_t K, hipStream_t stream) {
  clear_error();
  int rc;
  if ((rc = check_dtype(a.dtype)) || (rc = check_act_ext(a.act)) || (rc = q4_check_shape(a.M, N, K, a.group))) return rc;
  if (a.ws_bytes < 0) return fail(GP_ERR_INVALID_ARG, "workspace_bytes must be >= 0");
  if (a.ws_bytes && (rc = check16(a.ws, "workspace", true))) return rc;
  if (a.r && a.act != GP_ACT_NONE) return fail(GP_ERR_INVALID_ARG, "a residual is added without an activation only");
  for (int i = 0; i < a.sides; ++i) {
    const Q4Side& d = a.side[i];
    if ((rc = check16(d.wq, "wq", true)) || (rc = check16(d.s, "scales", true)) ||
        (rc = check16(d.z, "zeros", false)) || (rc = check16(d.b, "b", false)))
      return rc;
  }
  if ((rc = check16(a.r, "r", false))) return rc;
  if (a.M == 0) return GP_OK;
  if ((rc = check16(a.x, "x", true)) || (rc = check16(a.out, "out", true))) return rc;
  if (meet(a.out, a.M * N, a.x, a.M * K)) return fail(GP_ERR_INVALID_ARG, "out must not overlap x");
  if (a.r != a.out && meet(a.out, a.M * N, a.r, a.M * N))
    return fail(GP_ERR_INVALID_ARG, "out may be r, but not overlap it otherwise");
  if (meet(a.ws, a.ws_bytes / 2, a.x, a.M * K) || meet(a.ws, a.ws_bytes / 2, a.out, a.M * N) ||
      meet(a.ws, a.ws_bytes / 2, a.r, a.M * N))
    return fail(GP_ERR_INVALID_ARG, "the workspace must not overlap x, r or out");
  const int64_t scales = (K + a.group - 1) / a.group * N;
  for (int i = 0; i < a.sides; ++i) {
    const Q4Side& d = a.side[i];
    auto meets = [&](const void* p, int64_t n) {
      return meet(p, n, d.wq, K / 4 * N) || meet(p, n, d.s, scales) || meet(p, n, d.z, scales) || meet(p, n, d.b, N);
    };
    if (meets(a.out, a.M * N)) return fail(GP_ERR_INVALID_ARG, "out must not overlap a weight, its scales, zeros or b");
    if (meets(a.ws, a.ws_bytes / 2))
      return fail(GP_ERR_INVALID_ARG, "the workspace must not overlap a weight, its scales, zeros or b");
  }
  int dev = 0, ncu = 0;
  if ((rc = current_device_info(&dev, &ncu))) return rc;
  Q4Args b = a;
  b.N = (int)N;
  b.K = (int)K;
  const hipError_t e = q4_launch(b, ncu, stream);
  return e == hipSuccess ? GP_OK : fail_hip(e, "q4 launch");
}

// Whether `n` bytes at a and `m` at b have memory in common (NULL has none).
bool meet_bytes(const void* a, int64_t n, const void* b, int64_t m) {
  return a && b && (uintptr_t)a < (uintptr_t)b + (uintptr_t)m && (uintptr_t)b < (uintptr_t)a + (uintptr_t)n;
}

int64_t i8_packed(int64_t N, int64_t K) { return (N + 15) / 16 * ((K + 63) / 64) * 1024; }

int i8_check_weight(int64_t N, int64_t K, const char* n, const char* k) {
  if (K < 16 || K % 16 || K > kI8MaxK)
    return fail(GP_ERR_SHAPE, "%s must be a multiple of 16 in [16, %lld] (got %lld)", k, (long long)kI8MaxK, (long long)K);
  if (N < 1 || N > kQ4MaxDim) return fail(GP_ERR_SHAPE, "%s must be in [1, %lld] (got %lld)", n, (long long)kQ4MaxDim, (long long)N);
  if (i8_packed(N, K) >= (int64_t(1) << 31)) return fail(GP_ERR_SHAPE, "a packed weight must be smaller than 2 GiB");
  return GP_OK;
}

// Scales: 32-bit values of their own alignment.
int check4(const void* p, const char* name, bool needed) {
  if (!p) return needed ? fail(GP_ERR_INVALID_ARG, "%s is NULL", name) : GP_OK;
  if ((uintptr_t)p % 4) return fail(GP_ERR_ALIGN, "%s must be 4-byte aligned", name);
  return GP_OK;
}

int i8_check_shape(int64_t M, int64_t N, int64_t K) {
  int rc = check_rows(M);
  if (rc || (rc = i8_check_weight(N, K, "N", "K"))) return rc;
  if (M > (int64_t(1) << 21)) return fail(GP_ERR_SHAPE, "M must be at most 2097152 (got %lld)", (long long)M);
  return GP_OK;
}

// a.x is x, 16-bit or (a.xs given) bytes.
int i8_run(I8Args a, int64_t N, int64_t K, int64_t ws_bytes, hipStream_t stream) {
  clear_error();
  int rc;
  if ((rc = check_dtype(a.dtype)) || (rc = check_act_ext(a.act)) || (rc = i8_check_shape(a.M, N, K))) return rc;
  if (ws_bytes < 0) return fail(GP_ERR_INVALID_ARG, "workspace_bytes must be >= 0");
  if (ws_bytes && (rc = check16(a.ws, "workspace", true))) return rc;
  if (a.r && a.act != GP_ACT_NONE) return fail(GP_ERR_INVALID_ARG, "a residual is added without an activation only");
  for (int i = 0; i < a.sides; ++i) {
    const I8Side& d = a.side[i];
    if ((rc = check16(d.wq, "wq", true)) || (rc = check4(d.s, "w_scales", true)) || (rc = check16(d.b, "b", false)))
      return rc;
  }
  if ((rc = check4(a.xs, "x_scales", false)) || (rc = check16(a.r, "r", false))) return rc;
  if (a.M == 0) return GP_OK;
  if ((rc = check16(a.x, "x", true)) || (rc = check16(a.out, "out", true))) return rc;
  const int64_t out_bytes = a.M * N * 2, x_bytes = a.M * K * (a.xs ? 1 : 2);
  if (a.r != a.out && meet_bytes(a.out, out_bytes, a.r, out_bytes))
    return fail(GP_ERR_INVALID_ARG, "out may be r, but not overlap it otherwise");
  if (meet_bytes(a.ws, ws_bytes, a.out, out_bytes) || meet_bytes(a.ws, ws_bytes, a.r, out_bytes))
    return fail(GP_ERR_INVALID_ARG, "the workspace must not overlap r or out");
  auto meets = [&](const void* p, int64_t n) {
    if (meet_bytes(p, n, a.x, x_bytes) || meet_bytes(p, n, a.xs, a.M * 4)) return true;
    for (int i = 0; i < a.sides; ++i) {
      const I8Side& d = a.side[i];
      if (meet_bytes(p, n, d.wq, i8_packed(N, K)) || meet_bytes(p, n, d.s, N * 4) || meet_bytes(p, n, d.b, N * 2)) return true;
    }
    return false;
  };
  if (meets(a.out, out_bytes)) return fail(GP_ERR_INVALID_ARG, "out must not overlap x, a weight, scales or b");
  if (meets(a.ws, ws_bytes)) return fail(GP_ERR_INVALID_ARG, "the workspace must not overlap x, a weight, scales or b");
  int dev = 0, ncu = 0;
  if ((rc = current_device_info(&dev, &ncu))) return rc;
  a.N = (int)N;
  a.K = (int)K;
  const int64_t need = i8_workspace(a.M, a.N, a.K, !a.xs, a.sides, ncu);
  if (ws_bytes < need)
    return fail(GP_ERR_INVALID_ARG, "workspace_bytes must be at least %lld (got %lld)", (long long)need, (long long)ws_bytes);
  if (a.xs) a.xq = a.x;
  const hipError_t e = i8_launch(a, ncu, stream);
  return e == hipSuccess ? GP_OK : fail_hip(e, "i8 launch");
}

int experts_check_shape(int64_t T, int64_t H, int64_t F, int64_t E, int topk) {
  if (T < 0) return fail(GP_ERR_INVALID_ARG, "T must be >= 0 (got %lld)", (long long)T);
  int rc;
  if ((rc = i8_check_weight(F, H, "F", "H")) || (rc = i8_check_weight(H, F, "H", "F"))) return rc;
  if (E < 1 || E > kExpertsMaxE) return fail(GP_ERR_SHAPE, "E must be in [1, %d] (got %lld)", kExpertsMaxE, (long long)E);
  if (topk < 1 || topk > kExpertsMaxK) return fail(GP_ERR_SHAPE, "topk must be in [1, %d] (got %d)", kExpertsMaxK, topk);
  if (T > (int64_t(1) << 21) || T * H >= (int64_t(1) << 31))
    return fail(GP_ERR_SHAPE, "T must be at most 2097152, and T * H below 2^31 (got %lld, %lld)", (long long)T, (long long)H);
  return GP_OK;
}

int experts_run(const ExpertsArgs& a, int64_t ws_bytes, hipStream_t stream) {
  int rc;
  if ((rc = check_dtype(a.dtype)) || (rc = check_act_ext(a.act))) return rc;
  if (ws_bytes < 0) return fail(GP_ERR_INVALID_ARG, "workspace_bytes must be >= 0");
  if (ws_bytes && (rc = check16(a.ws, "workspace", true))) return rc;
  if ((rc = check16(a.wg, "wq_g", true)) || (rc = check4(a.sg, "w_scales_g", true)) || (rc = check16(a.wu, "wq_u", true)) ||
      (rc = check4(a.su, "w_scales_u", true)) || (rc = check16(a.wd, "wq_d", true)) ||
      (rc = check4(a.sd, "w_scales_d", true)) || (rc = check16(a.r, "r", false)))
    return rc;
  if (a.T == 0) return GP_OK;
  if ((rc = check16(a.x, "x", true)) || (rc = check4(a.ids, "ids", true)) || (rc = check4(a.weights, "weights", true)) ||
      (rc = check16(a.out, "out", true)))
    return rc;
  const int64_t bytes = a.T * a.H * 2, P = a.T * a.topk;
  if (a.r != a.out && meet_bytes(a.out, bytes, a.r, bytes))
    return fail(GP_ERR_INVALID_ARG, "out may be r, but not overlap it otherwise");
  if (meet_bytes(a.ws, ws_bytes, a.out, bytes) || meet_bytes(a.ws, ws_bytes, a.r, bytes))
    return fail(GP_ERR_INVALID_ARG, "the workspace must not overlap r or out");
  auto meets = [&](const void* p, int64_t n) {
    const int64_t E = a.E, up = E * i8_packed(a.F, a.H), down = E * i8_packed(a.H, a.F);
    return meet_bytes(p, n, a.x, bytes) || meet_bytes(p, n, a.ids, P * 4) || meet_bytes(p, n, a.weights, P * 4) ||
           meet_bytes(p, n, a.wg, up) || meet_bytes(p, n, a.sg, E * a.F * 4) || meet_bytes(p, n, a.wu, up) ||
           meet_bytes(p, n, a.su, E * a.F * 4) || meet_bytes(p, n, a.wd, down) || meet_bytes(p, n, a.sd, E * a.H * 4);
  };
  if (meets(a.out, bytes)) return fail(GP_ERR_INVALID_ARG, "out must not overlap x, ids, weights, an expert's weight or scales");
  if (meets(a.ws, ws_bytes))
    return fail(GP_ERR_INVALID_ARG, "the workspace must not overlap x, ids, weights, an expert's weight or scales");
  int dev = 0, ncu = 0;
  if ((rc = current_device_info(&dev, &ncu))) return rc;
  const int64_t need = i8_experts_workspace(a.T, a.H, a.F, a.E, a.topk, ncu);
  if (ws_bytes < need)
    return fail(GP_ERR_INVALID_ARG, "workspace_bytes must be at least %lld (got %lld)", (long long)need, (long long)ws_bytes);
  const hipError_t e = i8_experts_launch(a, ncu, stream);
  return e == hipSuccess ? GP_OK : fail_hip(e, "i8 experts launch");
}

}  // namespace
}  // namespace gp

using namespace gp;

extern "C" {

int gp_residual_norm_out(int64_t M, int64_t D, const void* x, const void* y, int post, const void* post_gamma,
                         const void* post_beta, float post_eps, const void* gate, int64_t gate_rows, int gate_act,
                         float scale, int pre, const void* gamma, const void* beta, float eps, void* h, void* out,
                         int dtype, void* stream) {
  clear_error();
  int rc;
  if ((rc = check_dtype(dtype)) || (rc = check_rows(M))) return rc;
  if (D < 1 || D > kNormMaxDim)
    return fail(GP_ERR_SHAPE, "D must be in [1, %lld] (got %lld)", (long long)kNormMaxDim, (long long)D);
  if ((rc = check_norm(post, post_gamma, post_beta, post_eps, "post")) ||
      (rc = check_norm(pre, gamma, beta, eps, "pre")))
    return rc;
  if (gate) {
    if ((rc = check_act_ext(gate_act))) return rc;
    if (M > 0 && (gate_rows < 1 || M % gate_rows))
      return fail(GP_ERR_SHAPE, "gate_rows must be a divisor of M (%lld rows, got %lld)", (long long)M,
                  (long long)gate_rows);
  }
  if (!std::isfinite(scale)) return fail(GP_ERR_INVALID_ARG, "scale must be finite");
  if (M == 0) return GP_OK;
  if (!x) return fail(GP_ERR_INVALID_ARG, "x is NULL");
  if (!y && (post != GP_NORM_NONE || gate))
    return fail(GP_ERR_INVALID_ARG, "without y there is no post norm and no gate");
  if (pre != GP_NORM_NONE ? !out : out != nullptr)
    return fail(GP_ERR_INVALID_ARG, "out must be given if there is a pre norm, and only then");
  if (!h && !out) return fail(GP_ERR_INVALID_ARG, "neither h nor out is given");
  if (h && h == out) return fail(GP_ERR_INVALID_ARG, "h and out must not be the same memory");
  const void* all[] = {x, y, post_gamma, post_beta, gate, gamma, beta, h, out};
  for (const void* p : all)
    if ((uintptr_t)p % 2) return fail(GP_ERR_ALIGN, "every tensor must be 2-byte aligned");
  if (meet(h, M * D, out, M * D)) return fail(GP_ERR_INVALID_ARG, "h and out must not overlap");
  for (const void* o : {(const void*)h, (const void*)out}) {
    for (const void* p : {x, y})
      if (o != p && meet(o, M * D, p, M * D))
        return fail(GP_ERR_INVALID_ARG, "h and out may be x or y, but not overlap them otherwise");
    if ((o != gate || gate_rows != M) && meet(o, M * D, gate, gate_rows * D))
      return fail(GP_ERR_INVALID_ARG, "h and out may be a gate of M rows, but not overlap it otherwise");
    for (const void* p : {post_gamma, post_beta, gamma, beta})
      if (meet(o, M * D, p, D)) return fail(GP_ERR_INVALID_ARG, "h and out must not overlap a gamma or beta");
  }
  int dev = 0, ncu = 0;
  if ((rc = current_device_info(&dev, &ncu))) return rc;
  const ResidualNormArgs a{M,     D,    x,   y,     post, post_gamma, post_beta, post_eps, gate, gate_rows, gate_act,
                           scale, pre,  gamma, beta, eps,  h,          out,       dtype};
  const hipError_t e = residual_norm_launch(a, ncu, (hipStream_t)stream);
  return e == hipSuccess ? GP_OK : fail_hip(e, "residual_norm launch");
}

int64_t gp_q4_workspace_bytes(int64_t M, int64_t N, int64_t K, int group, int weights) {
  clear_error();
  int rc = q4_check_shape(M, N, K, group);
  if (rc) return rc;
  if (weights != 1 && weights != 2) return fail(GP_ERR_INVALID_ARG, "weights must be 1 or 2 (got %d)", weights);
  if (M == 0) return 0;
  int dev = 0, ncu = 0;
  if ((rc = current_device_info(&dev, &ncu))) return rc;
  return q4_workspace(M, (int)N, (int)K, group, weights, ncu);
}

int gp_q4_gemm_out(int64_t M, int64_t N, int64_t K, int group, const void* x, const void* wq, const void* scales,
                   const void* zeros, const void* b, const void* r, int act, void* out, void* workspace,
                   int64_t workspace_bytes, int dtype, void* stream) {
  const Q4Args a{M, 0, 0, group, 1, x, {{wq, scales, zeros, b}, {}}, r, act, out, dtype, workspace, workspace_bytes};
  return q4_run(a, N, K, (hipStream_t)stream);
}

int gp_q4_gated_out(int64_t M, int64_t N, int64_t K, int group, const void* x, const void* wq_g, const void* scales_g,
                    const void* zeros_g, const void* b_g, const void* wq_u, const void* scales_u, const void* zeros_u,
                    const void* b_u, int act, void* out, void* workspace, int64_t workspace_bytes, int dtype,
                    void* stream) {
  const Q4Args a{M,   0,  0,       group, 2, x, {{wq_g, scales_g, zeros_g, b_g}, {wq_u, scales_u, zeros_u, b_u}},
                 nullptr, act, out, dtype, workspace, workspace_bytes};
  return q4_run(a, N, K, (hipStream_t)stream);
}

int64_t gp_i8_workspace_bytes(int64_t M, int64_t N, int64_t K, int x_int8, int weights) {
  clear_error();
  int rc = i8_check_shape(M, N, K);
  if (rc) return rc;
  if (x_int8 != 0 && x_int8 != 1) return fail(GP_ERR_INVALID_ARG, "x_int8 must be 0 or 1 (got %d)", x_int8);
  if (weights != 1 && weights != 2) return fail(GP_ERR_INVALID_ARG, "weights must be 1 or 2 (got %d)", weights);
  if (M == 0) return 0;
  int dev = 0, ncu = 0;
  if ((rc = current_device_info(&dev, &ncu))) return rc;
  return i8_workspace(M, (int)N, (int)K, !x_int8, weights, ncu);
}

int gp_i8_gemm_out(int64_t M, int64_t N, int64_t K, const void* x, const void* x_scales, const void* wq,
                   const void* w_scales, const void* b, const void* r, int act, void* out, void* workspace,
                   int64_t workspace_bytes, int dtype, void* stream) {
  const I8Args a{M, 0, 0, 1, x, nullptr, (const float*)x_scales, {{wq, (const float*)w_scales, b}, {}}, r, act, out,
                 dtype, workspace, nullptr};
  return i8_run(a, N, K, workspace_bytes, (hipStream_t)stream);
}

int gp_i8_gated_out(int64_t M, int64_t N, int64_t K, const void* x, const void* x_scales, const void* wq_g,
                    const void* w_scales_g, const void* b_g, const void* wq_u, const void* w_scales_u, const void* b_u,
                    int act, void* out, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  const I8Args a{M, 0, 0, 2, x, nullptr, (const float*)x_scales,
                 {{wq_g, (const float*)w_scales_g, b_g}, {wq_u, (const float*)w_scales_u, b_u}}, nullptr, act, out,
                 dtype, workspace, nullptr};
  return i8_run(a, N, K, workspace_bytes, (hipStream_t)stream);
}

int gp_route_out(int64_t T, int64_t E, int k, const void* logits, const void* bias, int score, int groups,
                 int top_groups, int group_score, int renorm, float scale, void* weights, void* ids, int dtype,
                 void* stream) {
  clear_error();
  int rc;
  if (dtype != GP_DTYPE_F32 && (rc = check_dtype(dtype))) return rc;
  if (T < 0) return fail(GP_ERR_INVALID_ARG, "T must be >= 0 (got %lld)", (long long)T);
  if (T > (int64_t(1) << 30)) return fail(GP_ERR_SHAPE, "T too large (%lld)", (long long)T);
  if (E < 1 || E > kRouteMaxE) return fail(GP_ERR_SHAPE, "E must be in [1, %d] (got %lld)", kRouteMaxE, (long long)E);
  if (score != GP_SCORE_SOFTMAX && score != GP_SCORE_SIGMOID) return fail(GP_ERR_INVALID_ARG, "unknown score %d", score);
  if (group_score != GP_GROUP_MAX && group_score != GP_GROUP_TOP2)
    return fail(GP_ERR_INVALID_ARG, "unknown group score %d", group_score);
  if (groups < 1 || groups > kRouteMaxGroups || E % groups)
    return fail(GP_ERR_SHAPE, "groups must divide E and be at most %d (got %d)", kRouteMaxGroups, groups);
  if (top_groups < 1 || top_groups > groups)
    return fail(GP_ERR_SHAPE, "top_groups must be in [1, groups] (got %d)", top_groups);
  if (k < 1 || k > kRouteMaxK || k > E / groups * top_groups)
    return fail(GP_ERR_SHAPE, "k must be in [1, %d] and at most the experts of top_groups groups (got %d)", kRouteMaxK, k);
  if (renorm != 0 && renorm != 1) return fail(GP_ERR_INVALID_ARG, "renorm must be 0 or 1 (got %d)", renorm);
  if (!std::isfinite(scale)) return fail(GP_ERR_INVALID_ARG, "scale must be finite");
  if ((rc = check4(bias, "bias", false))) return rc;
  if (T == 0) return GP_OK;
  if (!logits) return fail(GP_ERR_INVALID_ARG, "logits is NULL");
  const int64_t size = dtype == GP_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)logits % size) return fail(GP_ERR_ALIGN, "logits must be aligned to its elements");
  if ((rc = check4(weights, "weights", true)) || (rc = check4(ids, "ids", true))) return rc;
  if (meet_bytes(weights, T * k * 4, ids, T * k * 4)) return fail(GP_ERR_INVALID_ARG, "weights and ids must not overlap");
  for (const void* o : {(const void*)weights, (const void*)ids})
    if (meet_bytes(o, T * k * 4, logits, T * E * size) || meet_bytes(o, T * k * 4, bias, E * 4))
      return fail(GP_ERR_INVALID_ARG, "weights and ids must not overlap the logits or the bias");
  int dev = 0, ncu = 0;
  if ((rc = current_device_info(&dev, &ncu))) return rc;
  const RouteExpertsArgs a{T,     (int)E, k, logits, (const float*)bias, score, groups, top_groups, group_score, renorm,
                    scale, (float*)weights, (int*)ids, dtype};
  const hipError_t e = route_experts_launch(a, (hipStream_t)stream);
  return e == hipSuccess ? GP_OK : fail_hip(e, "route launch");
}

int64_t gp_i8_experts_workspace_bytes(int64_t T, int64_t H, int64_t F, int64_t E, int topk) {
  clear_error();
  int rc = experts_check_shape(T, H, F, E, topk);
  if (rc) return rc;
  if (T == 0) return 0;
  int dev = 0, ncu = 0;
  if ((rc = current_device_info(&dev, &ncu))) return rc;
  return i8_experts_workspace(T, (int)H, (int)F, (int)E, topk, ncu);
}

int gp_i8_experts_out(int64_t T, int64_t H, int64_t F, int64_t E, int topk, const void* x, const void* ids,
                      const void* weights, const void* wq_g, const void* w_scales_g, const void* wq_u,
                      const void* w_scales_u, const void* wq_d, const void* w_scales_d, int act, const void* r, void* out,
                      void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  clear_error();
  const int rc = experts_check_shape(T, H, F, E, topk);
  if (rc) return rc;
  const ExpertsArgs a{T, (int)H, (int)F, (int)E, topk, x, (const int*)ids, (const float*)weights, wq_g, wq_u, wq_d,
                      (const float*)w_scales_g, (const float*)w_scales_u, (const float*)w_scales_d, act, r, out, dtype,
                      workspace};
  return experts_run(a, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
