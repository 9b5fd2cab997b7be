// fp8_blocks.cpp — matrices in e4m3 with block scales (orda_quant_fp8_blocks,
// orda_fp8_block_matmul of include/orda/orda.h). The calls queue their kernels
// and return; the scratch is the caller's.
#include "orda_host.h"

namespace orda {
namespace {

constexpr int64_t kMaxPitch = int64_t{1} << 20, kMaxStride = int64_t{1} << 22, kMaxRows = int64_t{1} << 30;

// A quantised matrix: its shape, pitch and scale strides.
void check_matrix(const orda_fp8_matrix& m, const char* what) {
  if (m.rows < 0 || m.cols < 0) fail(ORDA_ERR_INVALID, "%s has a negative shape", what);
  if (m.block_rows != 1 && m.block_rows != 128) fail(ORDA_ERR_INVALID, "%s: block_rows must be 1 or 128", what);
  if (m.rows > kMaxRows || m.cols > kMaxPitch) fail(ORDA_ERR_INVALID, "%s: at most 2^30 rows and 2^20 columns", what);
  if (m.rows == 0 || m.cols == 0) return;
  if (!m.codes || !m.scales) fail(ORDA_ERR_INVALID, "%s has a null data pointer", what);
  if (m.ld < m.cols || m.ld > kMaxPitch + 16) fail(ORDA_ERR_INVALID, "%s has a pitch out of range", what);
  if (m.scale_row < 0 || m.scale_col < 0 || m.scale_row > kMaxStride)
    fail(ORDA_ERR_INVALID, "%s has scale strides out of range", what);
}

bool in_place(const orda_fp8_matrix& m) {
  return m.ld % 16 == 0 && reinterpret_cast<uintptr_t>(m.codes) % 16 == 0;
}
int64_t packed_bytes(const orda_fp8_matrix& m) {
  if (m.rows == 0 || m.cols == 0 || in_place(m)) return 0;
  return (m.rows * ((m.cols + 15) / 16 * 16) + 255) / 256 * 256;
}

int64_t check_product(const orda_fp8_matrix& a, const orda_fp8_matrix& b) {
  check_matrix(a, "a");
  check_matrix(b, "b");
  if (a.block_rows != 1) fail(ORDA_ERR_INVALID, "a must have a scale for each row (block_rows 1)");
  if (b.block_rows != 128) fail(ORDA_ERR_INVALID, "b must have a scale for each 128 rows (block_rows 128)");
  if (a.cols != b.cols)
    fail(ORDA_ERR_INVALID, "a has %lld columns, b %lld", static_cast<long long>(a.cols), static_cast<long long>(b.cols));
  if (a.cols < 1) fail(ORDA_ERR_INVALID, "a and b must have columns");
  return packed_bytes(a) + packed_bytes(b);
}

}  // namespace
}  // namespace orda

using namespace orda;

extern "C" {

int32_t orda_quant_fp8_blocks(int32_t device, void* hip_stream, const orda_tensor* m, orda_fp8_matrix* out, char* err,
                              size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!m || !out) fail(ORDA_ERR_INVALID, "null argument");
    check_view(*m, "m");
    const DType t = to_dtype(m->dtype, "m");
    if (m->location != ORDA_DEVICE) fail(ORDA_ERR_INVALID, "m must be on the device");
    check_matrix(*out, "out");
    if (out->rows != m->rows || out->cols != m->cols) fail(ORDA_ERR_INVALID, "out must have the shape of m");
    if (m->rows == 0 || m->cols == 0) return;
    if (out->ld % 8 != 0 || reinterpret_cast<uintptr_t>(out->codes) % 8 != 0)
      fail(ORDA_ERR_INVALID, "out: codes must be 8-byte aligned with a pitch of whole 8s");
    const DeviceScope scope(device);
    const Fp8QuantArgs a{m->data, tensor_ld(*m), m->rows, m->cols, static_cast<uint8_t*>(out->codes), out->ld,
                         out->scales, out->scale_row, out->scale_col};
    hip_check(launch_fp8_quant(a, t, out->block_rows == 128, static_cast<hipStream_t>(hip_stream)), "fp8 quantisation");
  });
}

int32_t orda_fp8_block_matmul_workspace(const orda_fp8_matrix* a, const orda_fp8_matrix* b, int64_t* bytes, char* err,
                                        size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!a || !b || !bytes) fail(ORDA_ERR_INVALID, "null argument");
    *bytes = check_product(*a, *b);
  });
}

int32_t orda_fp8_block_matmul(int32_t device, void* hip_stream, const orda_fp8_matrix* a, const orda_fp8_matrix* b,
                              orda_tensor* out, void* workspace, int64_t workspace_bytes, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!a || !b || !out) fail(ORDA_ERR_INVALID, "null argument");
    const int64_t need = check_product(*a, *b);
    check_view(*out, "out");
    const DType t = to_dtype(out->dtype, "out");
    if (out->location != ORDA_DEVICE) fail(ORDA_ERR_INVALID, "out must be on the device");
    if (out->rows != a->rows || out->cols != b->rows)
      fail(ORDA_ERR_INVALID, "out must be [%lld, %lld]", static_cast<long long>(a->rows), static_cast<long long>(b->rows));
    if (a->rows == 0 || b->rows == 0) return;
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) fail(ORDA_ERR_INVALID, "workspace must be 256-byte aligned");
    if (workspace_bytes < need || (need > 0 && !workspace))
      fail(ORDA_ERR_INVALID, "workspace of %lld bytes, %lld needed", static_cast<long long>(workspace_bytes),
           static_cast<long long>(need));
    const DeviceScope scope(device);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    char* at = static_cast<char*>(workspace);
    auto operand = [&](const orda_fp8_matrix& m, int64_t& ld) -> const unsigned char* {
      const auto* codes = static_cast<const unsigned char*>(m.codes);
      ld = m.ld;
      if (in_place(m)) return codes;
      auto* p = reinterpret_cast<unsigned char*>(at);
      ld = (m.cols + 15) / 16 * 16;
      hip_check(launch_fp8_pack(codes, m.ld, m.rows, m.cols, p, ld, st), "fp8 codes");
      at += packed_bytes(m);
      return p;
    };
    Fp8MmArgs g{};
    g.a = operand(*a, g.lda);
    g.b = operand(*b, g.ldb);
    g.sa = a->scales;
    g.sa_row = a->scale_row;
    g.sa_col = a->scale_col;
    g.sb = b->scales;
    g.sb_row = b->scale_row;
    g.sb_col = b->scale_col;
    g.c = out->data;
    g.ldc = tensor_ld(*out);
    g.m = a->rows;
    g.n = b->rows;
    g.k = a->cols;
    hip_check(launch_fp8_mm(g, t, st), "fp8 product");
  });
}

}  // extern "C"
