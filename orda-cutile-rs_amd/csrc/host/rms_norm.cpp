// rms_norm.cpp — the root-mean-square norm and its gradients (orda_rms_norm_* of
// include/orda/orda.h). The calls queue their kernels and return; the scratch is
// the caller's.
#include <math.h>

#include "orda_host.h"

namespace orda {
namespace {

constexpr int64_t kMostRows = int64_t{1} << 30, kMostCols = int64_t{1} << 20;

DType check_matrix(const orda_tensor& t, const char* what) {
  check_view(t, what);
  const DType d = to_dtype(t.dtype, what);
  if (t.location != ORDA_DEVICE) fail(ORDA_ERR_INVALID, "%s must be on the device", what);
  if (t.rows > kMostRows || t.cols > kMostCols)
    fail(ORDA_ERR_INVALID, "%s: at most 2^30 rows and 2^20 columns", what);
  return d;
}
// A matrix of x's shape and type.
void check_like(const orda_tensor& t, const orda_tensor& x, DType d, const char* what) {
  if (check_matrix(t, what) != d) fail(ORDA_ERR_INVALID, "%s must have the rows' dtype", what);
  if (t.rows != x.rows || t.cols != x.cols)
    fail(ORDA_ERR_INVALID, "%s must be [%lld, %lld]", what, static_cast<long long>(x.rows), static_cast<long long>(x.cols));
}
struct Types {
  DType rows, weight;
};
Types check_args(const orda_rms_norm& a) {
  const DType d = check_matrix(a.x, "x");
  if (a.residual.data) check_like(a.residual, a.x, d, "residual");
  const DType w = check_matrix(a.weight, "weight");
  if (a.weight.rows != 1 || a.weight.cols != a.x.cols)
    fail(ORDA_ERR_INVALID, "weight must be [1, %lld]", static_cast<long long>(a.x.cols));
  if (!(a.eps >= 0.) || !isfinite(a.eps)) fail(ORDA_ERR_INVALID, "eps must be >= 0 and finite");
  if (!isfinite(a.weight_offset)) fail(ORDA_ERR_INVALID, "weight_offset must be finite");
  return {d, w};
}

NormArgs kernel_args(const orda_rms_norm& a, const Types& t, const orda_tensor* total) {
  NormArgs k{};
  k.x = a.x.data;
  k.ldx = tensor_ld(a.x);
  k.r = a.residual.data;
  k.ldr = tensor_ld(a.residual);
  k.w = a.weight.data;
  k.n = a.x.rows;
  k.h = a.x.cols;
  k.eps = a.eps;
  k.per_column = 1. / static_cast<double>(k.h);   // (not used where there is no column)
  k.offset = a.weight_offset;
  if (total && total->data) {
    check_like(*total, a.x, t.rows, "total");
    k.total = total->data;
    k.ldt = tensor_ld(*total);
  }
  return k;
}

}  // namespace
}  // namespace orda

using namespace orda;

extern "C" {

int32_t orda_rms_norm_forward(int32_t device, void* hip_stream, const orda_rms_norm* args, orda_tensor* total,
                              orda_tensor* out, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!args || !out) fail(ORDA_ERR_INVALID, "null argument");
    const Types t = check_args(*args);
    NormArgs k = kernel_args(*args, t, total);
    check_like(*out, args->x, t.rows, "out");
    if (k.n == 0 || k.h == 0) return;
    k.out = out->data;
    k.ldo = tensor_ld(*out);
    const DeviceScope scope(device);
    hip_check(launch_norm(k, t.rows, t.weight, static_cast<hipStream_t>(hip_stream)), "norm");
  });
}

int32_t orda_rms_norm_fp8(int32_t device, void* hip_stream, const orda_rms_norm* args, orda_tensor* total,
                          orda_fp8_matrix* out, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!args || !out) fail(ORDA_ERR_INVALID, "null argument");
    const Types t = check_args(*args);
    NormArgs k = kernel_args(*args, t, total);
    check_fp8_matrix(*out, "out");
    if (out->block_rows != 1) fail(ORDA_ERR_INVALID, "out must have a scale for each row (block_rows 1)");
    if (out->rows != k.n || out->cols != k.h) fail(ORDA_ERR_INVALID, "out must have the shape of x");
    if (k.n == 0 || k.h == 0) return;
    if (out->ld % 8 != 0 || reinterpret_cast<uintptr_t>(out->codes) % 8 != 0)
      fail(ORDA_ERR_INVALID, "out: codes must be 8-byte aligned with a pitch of whole 8s");
    k.codes = static_cast<uint8_t*>(out->codes);
    k.ldc = out->ld;
    k.scales = out->scales;
    k.scale_row = out->scale_row;
    k.scale_col = out->scale_col;
    const DeviceScope scope(device);
    hip_check(launch_norm(k, t.rows, t.weight, static_cast<hipStream_t>(hip_stream)), "norm");
  });
}

int32_t orda_rms_norm_backward_workspace(int64_t n, int64_t h, int64_t* bytes, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!bytes) fail(ORDA_ERR_INVALID, "null argument");
    if (n < 0 || h < 0 || n > kMostRows || h > kMostCols)
      fail(ORDA_ERR_INVALID, "x: at most 2^30 rows and 2^20 columns");
    *bytes = norm_grad_scratch(n, h);
  });
}

int32_t orda_rms_norm_backward(int32_t device, void* hip_stream, const orda_rms_norm* args, const orda_tensor* grad_out,
                               const orda_tensor* grad_total, orda_tensor* grad_x, orda_tensor* grad_weight,
                               void* workspace, int64_t workspace_bytes, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!args || !grad_out) fail(ORDA_ERR_INVALID, "null argument");
    const Types t = check_args(*args);
    if (args->residual.data) fail(ORDA_ERR_INVALID, "the backward's x is the sum: no residual");
    check_like(*grad_out, args->x, t.rows, "grad_out");
    NormGradArgs k{};
    k.g = grad_out->data;
    k.ldg = tensor_ld(*grad_out);
    k.t = args->x.data;
    k.ldt = tensor_ld(args->x);
    if (grad_total && grad_total->data) {
      check_like(*grad_total, args->x, t.rows, "grad_total");
      k.gt = grad_total->data;
      k.ldgt = tensor_ld(*grad_total);
    }
    k.w = args->weight.data;
    k.n = args->x.rows;
    k.h = args->x.cols;
    k.eps = args->eps;
    k.per_column = 1. / static_cast<double>(k.h);
    k.offset = args->weight_offset;
    if (grad_x && grad_x->data) {
      check_like(*grad_x, args->x, t.rows, "grad_x");
      k.dx = grad_x->data;
      k.ldd = tensor_ld(*grad_x);
    }
    if (grad_weight && grad_weight->data) {
      if (check_matrix(*grad_weight, "grad_weight") != t.weight)
        fail(ORDA_ERR_INVALID, "grad_weight must have the weight's dtype");
      if (grad_weight->rows != 1 || grad_weight->cols != k.h)
        fail(ORDA_ERR_INVALID, "grad_weight must be [1, %lld]", static_cast<long long>(k.h));
      k.dw = grad_weight->data;
    }
    if (k.h == 0 || (!k.dx && !k.dw)) return;
    const int64_t need = norm_grad_scratch(k.n, k.h);
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) fail(ORDA_ERR_INVALID, "workspace must be 256-byte aligned");
    if (workspace_bytes < need || (need > 0 && !workspace))
      fail(ORDA_ERR_INVALID, "workspace of %lld bytes, %lld needed", static_cast<long long>(workspace_bytes),
           static_cast<long long>(need));
    k.ws = workspace;
    const DeviceScope scope(device);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (k.n == 0) {
      if (k.dw) hip_check(launch_zero_rows(t.weight, k.dw, k.h, 1, k.h, st), "norm gradient");
      return;
    }
    hip_check(launch_norm_grad(k, t.rows, t.weight, st), "norm gradient");
  });
}

}  // extern "C"
