// orda_host.h — internal host-side declarations of liborda_hip.so.
#pragma once

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <exception>
#include <string>
#include <vector>

#include "../../../include/orda/orda.h"
#include "../kernels/orda_kernels.h"

namespace orda {

struct ChunkPlan {
  int64_t chunk_size;
  int64_t num_chunks;
};

int64_t ceil_div(int64_t a, int64_t b);
int64_t chunks_from_raw(double raw);
ChunkPlan resolve_chunk_size(int64_t bt, bool fixed, int64_t fixed_rows, bool has_v, int64_t v,
                             bool has_max_chunks, int64_t max_chunks);
int64_t default_max_chunks_limit(int64_t bt);
std::vector<int64_t> chunk_doubling_schedule(int64_t bt, int64_t start, int64_t limit);

// Error carried to the C ABI boundary.
struct Error {
  int32_t status;
  std::string msg;
};

[[noreturn]] inline void fail(int32_t status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  throw Error{status, buf};
}

inline void hip_check(hipError_t e, const char* what) {
  if (e == hipSuccess) return;
  (void)hipGetLastError();
  if (e == hipErrorOutOfMemory) fail(ORDA_ERR_OOM, "%s: device out of memory", what);
  fail(ORDA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

inline void copy_err(const Error& e, char* err, size_t len) {
  if (!err || !len) return;
  snprintf(err, len, "%s", e.msg.c_str());
}

inline int64_t round8(int64_t x) { return (x + 7) / 8 * 8; }
inline int64_t round64(int64_t x) { return (x + 63) / 64 * 64; }

// Pitch of the logits staging rows: V rounded up to 64 elements, so that every
// row starts on a 128-byte line (the backward GEMMs read these rows in
// 128-byte K-slabs: at V = 50257 a pitch of round8(V) put every slab across two
// lines, grad_hidden 0.524 of peak against 0.60, the row pass 0.65 against
// 0.75). fp32 rows: plus 64 when that is a multiple of 1024, so that rows (and
// the many row streams the row pass and the GEMMs walk in step) do not sit a
// power of two apart. bf16 rows: further up to 64 past a multiple of 1024,
// which measured the bf16 row pass (BT = 8192, paired rows, TB/s, two passes)
// at V = 151936 5.9 against 5.0, at 50257 6.0 against 5.7, at 100000 and 128256
// 1-2 % faster, at 32000 and 200064 1-3 % slower, elsewhere equal; the
// backward GEMMs equal. (fp32 rows at V = 32000: the row pass 1.5 % slower,
// so fp32 keeps the first rule.)
inline int64_t logits_pitch(int64_t v, DType lt) {
  int64_t p = round64(v);
  if (lt == DType::BF16) {
    while (p % 1024 != 64) p += 64;
    return p;
  }
  return p % 1024 == 0 ? p + 64 : p;
}

inline int64_t tensor_ld(const orda_tensor& t) { return t.ld ? t.ld : t.cols; }

inline DType to_dtype(int32_t d, const char* what) {
  if (d == ORDA_F32) return DType::F32;
  if (d == ORDA_BF16) return DType::BF16;
  fail(ORDA_ERR_INVALID, "%s must be float32 or bfloat16", what);
}

// The checks every caller tensor passes before any kernel reads it: a
// non-negative shape, a data pointer when it has elements, ld >= cols.
inline void check_view(const orda_tensor& t, const char* what) {
  if (t.rows < 0 || t.cols < 0) fail(ORDA_ERR_INVALID, "%s has a negative shape", what);
  if (t.rows > 0 && t.cols > 0 && !t.data) fail(ORDA_ERR_INVALID, "%s has a null data pointer", what);
  if (tensor_ld(t) < t.cols) fail(ORDA_ERR_INVALID, "%s has ld < cols", what);
}

// A C entry point's body: no exception leaves it.
template <class F>
int32_t guarded(char* err, size_t err_len, F&& f) {
  try {
    f();
    return ORDA_OK;
  } catch (const Error& e) {
    copy_err(e, err, err_len);
    return e.status;
  } catch (const std::exception& e) {
    copy_err(Error{ORDA_ERR_INTERNAL, e.what()}, err, err_len);
    return ORDA_ERR_INTERNAL;
  }
}

// The calling thread's current device for the scope of a call.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    hip_check(hipGetDevice(&old_), "hipGetDevice");
    if (old_ != device) hip_check(hipSetDevice(device), "hipSetDevice");
    else old_ = -1;
  }
  ~DeviceScope() {
    if (old_ >= 0) (void)hipSetDevice(old_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int old_ = -1;
};

// Caller-provided scratch of the chunk-launcher entry point, for at most
// max_rows rows a call.
struct SlotScratch {
  int64_t max_rows;
  void* p;
  int64_t bytes;
};

// kl_ce_on_logits_chunk (src/cuda/launch.rs:51-158) behind both C entry
// points; throws Error. With sc every tensor must be on the device and
// nothing is allocated.
void kl_ce_slot(orda_ctx* c, const orda_tensor* logits_chunk, const int32_t* targets,
                int32_t targets_location, int64_t n_rows, float inv_t, float kl_grad_scale,
                float t_sq, float student_ce_weight, float teacher_ce_weight,
                float label_smoothing, int32_t ignore_index, int32_t student_only,
                int32_t compute_kl, orda_tensor* grad_kl_student, orda_tensor* kl_per_row,
                orda_tensor* grad_ce, orda_tensor* ce_loss, const SlotScratch* sc);

int32_t ctx_device(const orda_ctx* c);

// Looks up, once per device, the device address of the no-allocation entry
// point's scratch array (call with that device current). Returns a HIP error.
hipError_t noalloc_scratch_init(int device);

}  // namespace orda
