// sample.cpp — tokens drawn from logits (orda_sample_tokens of
// include/orda/orda.h). The calls queue their kernels and return; the scratch is
// the caller's.
#include <math.h>

#include "orda_host.h"

namespace orda {
namespace {

constexpr int64_t kMost = int64_t{1} << 20;

void check_shape(int64_t n, int64_t v) {
  if (n < 0 || v < 0) fail(ORDA_ERR_INVALID, "logits has a negative shape");
  if (n > kMost || v > kMost) fail(ORDA_ERR_INVALID, "logits: at most 2^20 rows and columns");
}

}  // namespace
}  // namespace orda

using namespace orda;

extern "C" {

int32_t orda_sample_tokens_workspace(int64_t n, int64_t v, int32_t dtype, int64_t* bytes, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!bytes) fail(ORDA_ERR_INVALID, "null argument");
    check_shape(n, v);
    int64_t tops, firsts, tails;
    *bytes = sample_scratch(to_dtype(dtype, "logits"), n, v, &tops, &firsts, &tails);
  });
}

int32_t orda_sample_tokens(int32_t device, void* hip_stream, const orda_sampling* args, int64_t* tokens, float* logprobs,
                           void* workspace, int64_t workspace_bytes, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!args) fail(ORDA_ERR_INVALID, "null argument");
    const orda_tensor& x = args->logits;
    check_view(x, "logits");
    const DType t = to_dtype(x.dtype, "logits");
    if (x.location != ORDA_DEVICE) fail(ORDA_ERR_INVALID, "logits must be on the device");
    check_shape(x.rows, x.cols);
    if (!args->temperatures && !(args->temperature >= 0.f && isfinite(args->temperature)))
      fail(ORDA_ERR_INVALID, "temperature must be >= 0 and finite");
    if (!args->top_ps && !(args->top_p >= 0.f && args->top_p <= 1.f))
      fail(ORDA_ERR_INVALID, "top_p must be in [0, 1]");
    if (!args->min_ps && !(args->min_p >= 0.f && args->min_p <= 1.f))
      fail(ORDA_ERR_INVALID, "min_p must be in [0, 1]");
    if (x.rows == 0) return;
    if (x.cols == 0) fail(ORDA_ERR_INVALID, "logits must have columns");
    if (!args->uniform || !tokens) fail(ORDA_ERR_INVALID, "null argument");
    int64_t tops, firsts, tails;
    const int64_t need = sample_scratch(t, x.rows, x.cols, &tops, &firsts, &tails);
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) fail(ORDA_ERR_INVALID, "workspace must be 256-byte aligned");
    if (workspace_bytes < need || !workspace)
      fail(ORDA_ERR_INVALID, "workspace of %lld bytes, %lld needed", static_cast<long long>(workspace_bytes),
           static_cast<long long>(need));
    SampleArgs a{};
    a.x = x.data;
    a.n = x.rows;
    a.v = x.cols;
    a.ldx = tensor_ld(x);
    a.u = args->uniform;
    a.t = args->temperatures;
    a.p = args->top_ps;
    a.m = args->min_ps;
    a.k = args->top_ks;
    a.t1 = args->temperature;
    a.p1 = args->top_p;
    a.m1 = args->min_p;
    a.k1 = args->top_k;
    a.token = tokens;
    a.logprob = logprobs;
    a.n64 = ceil_div(x.cols, 64);
    a.n1024 = ceil_div(x.cols, 1024);
    char* ws = static_cast<char*>(workspace);
    a.masses = reinterpret_cast<double*>(ws);
    a.tops = reinterpret_cast<uint32_t*>(ws + tops);
    a.firsts = reinterpret_cast<uint32_t*>(ws + firsts);
    a.tails = ws + tails;
    const DeviceScope scope(device);
    hip_check(launch_sample(a, t, static_cast<hipStream_t>(hip_stream)), "drawing tokens");
  });
}

}  // extern "C"
