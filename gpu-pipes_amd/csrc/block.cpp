// C ABI of the operators around a language model's feed-forward half: the norms
// with the residual (gp_residual_norm_out) and the products with 4-bit weights
// (gp_q4_gemm_out, gp_q4_gated_out).  Argument checks and dispatch; the kernels
// are in residual_norm.hip and q4.hip.
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

}  // extern "C"
