// embed.cpp — the embedding and its gradient (orda_embedding* of
// include/orda/orda.h). The calls queue their kernels and return; the scratch is
// the caller's.
#include "orda_host.h"

namespace orda {
namespace {

void check_ids(const void* ids, int32_t ids_bytes, int64_t n) {
  if (ids_bytes != 4 && ids_bytes != 8) fail(ORDA_ERR_INVALID, "ids must be int32 or int64");
  if (n < 0 || n > (int64_t{1} << 30)) fail(ORDA_ERR_INVALID, "at most 2^30 ids");
  if (n > 0 && !ids) fail(ORDA_ERR_INVALID, "ids have a null data pointer");
}

DType check_rows(const orda_tensor& t, const char* what) {
  check_view(t, what);
  const DType d = to_dtype(t.dtype, what);
  if (t.location != ORDA_DEVICE) fail(ORDA_ERR_INVALID, "%s must be on the device", what);
  if (t.rows > (int64_t{1} << 30) || t.cols > (int64_t{1} << 20))
    fail(ORDA_ERR_INVALID, "%s: at most 2^30 rows and 2^20 columns", what);
  return d;
}

}  // namespace
}  // namespace orda

using namespace orda;

extern "C" {

int32_t orda_embedding(int32_t device, void* hip_stream, const void* ids, int32_t ids_bytes, int64_t n,
                       const orda_tensor* weight, float scale, orda_tensor* out, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!weight || !out) fail(ORDA_ERR_INVALID, "null argument");
    check_ids(ids, ids_bytes, n);
    const DType t = check_rows(*weight, "weight");
    if (check_rows(*out, "out") != t) fail(ORDA_ERR_INVALID, "out must have the weight's dtype");
    if (out->rows != n || out->cols != weight->cols)
      fail(ORDA_ERR_INVALID, "out must be [%lld, %lld]", static_cast<long long>(n), static_cast<long long>(weight->cols));
    if (n == 0 || weight->cols == 0) return;
    const DeviceScope scope(device);
    hip_check(launch_embedding(t, ids, ids_bytes == 8, n, weight->data, tensor_ld(*weight), weight->rows, weight->cols,
                               scale, out->data, tensor_ld(*out), static_cast<hipStream_t>(hip_stream)),
              "embedding");
  });
}

int32_t orda_embedding_backward_workspace(int64_t n, int64_t rows, int64_t cols, int32_t grad_dtype, int64_t* bytes,
                                          char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!bytes) fail(ORDA_ERR_INVALID, "null argument");
    const orda_tensor t{nullptr, 0, 0, 0, grad_dtype, ORDA_DEVICE};
    const DType d = check_rows(t, "grad");
    check_ids(bytes, 8, n);
    if (rows < 0 || cols < 0 || rows > (int64_t{1} << 30) || cols > (int64_t{1} << 20))
      fail(ORDA_ERR_INVALID, "out: at most 2^30 rows and 2^20 columns");
    *bytes = embed_scratch(d, n, rows, cols).bytes;
  });
}

int32_t orda_embedding_backward(int32_t device, void* hip_stream, const void* ids, int32_t ids_bytes, int64_t n,
                                const orda_tensor* grad, int64_t padding_idx, float scale, int32_t accumulate,
                                orda_tensor* out, void* workspace, int64_t workspace_bytes, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!grad || !out) fail(ORDA_ERR_INVALID, "null argument");
    check_ids(ids, ids_bytes, n);
    const DType gt = check_rows(*grad, "grad"), ot = check_rows(*out, "out");
    if (grad->rows != n || grad->cols != out->cols)
      fail(ORDA_ERR_INVALID, "grad must be [%lld, %lld]", static_cast<long long>(n), static_cast<long long>(out->cols));
    if (out->rows == 0 || out->cols == 0 || (n == 0 && accumulate)) return;
    const EmbedScratch s = embed_scratch(gt, n, out->rows, out->cols);
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) fail(ORDA_ERR_INVALID, "workspace must be 256-byte aligned");
    if (workspace_bytes < s.bytes || (s.bytes > 0 && !workspace))
      fail(ORDA_ERR_INVALID, "workspace of %lld bytes, %lld needed", static_cast<long long>(workspace_bytes),
           static_cast<long long>(s.bytes));
    const DeviceScope scope(device);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    EmbedGradArgs a{};
    EmbedFill fill{};
    if (!accumulate) fill = embed_fill(ot, out->data, tensor_ld(*out), out->rows, out->cols);
    hip_check(launch_embed_sort(ids, ids_bytes == 8, n, out->rows, padding_idx, workspace, s, fill, &a.keys, &a.vals, st),
              "embedding gradient sort");
    a.n = n;
    a.v = out->rows;
    a.h = out->cols;
    a.grad = grad->data;
    a.ldg = tensor_ld(*grad);
    a.out = out->data;
    a.ldo = tensor_ld(*out);
    a.scale = scale;
    a.accumulate = accumulate != 0;
    a.chunk = s.chunk;
    a.chunks = s.chunks;
    a.slabs = s.slabs;
    a.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + s.parts);
    a.ldp = s.ldp;
    hip_check(launch_embed_grad(a, gt, ot, st), "embedding gradient");
  });
}

}  // extern "C"
