// C ABI of the operators around a language model's feed-forward half: the norms
// with the residual (gp_residual_norm_out).  Argument checks and dispatch; the
// kernels are in residual_norm.hip.
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
  int dev = 0, ncu = 0;
  if ((rc = current_device_info(&dev, &ncu))) return rc;
  const ResidualNormArgs a{M,     D,    x,   y,     post, post_gamma, post_beta, post_eps, gate, gate_rows, gate_act,
                           scale, pre,  gamma, beta, eps,  h,          out,       dtype};
  const hipError_t e = residual_norm_launch(a, ncu, (hipStream_t)stream);
  return e == hipSuccess ? GP_OK : fail_hip(e, "residual_norm launch");
}

}  // extern "C"
