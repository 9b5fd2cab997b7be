// gradients.cpp — the norm of many gradients and their clipping
// (orda_gradient_norm, orda_clip_gradients of include/orda/orda.h). The calls queue
// their kernels and return; the scratch is the caller's.
#include <math.h>

#include <algorithm>
#include <vector>

#include "orda_host.h"

namespace orda {
namespace {

constexpr int64_t kMostGradients = int64_t{1} << 20, kMostValues = int64_t{1} << 40;

// One row where nothing lies between the rows.
GradPart part_of(const orda_tensor& src, const orda_tensor& dst) {
  GradPart p{};
  p.src = src.data;
  p.dst = dst.data;
  p.rows = src.rows;
  p.cols = src.cols;
  p.lds = tensor_ld(src);
  p.ldd = tensor_ld(dst);
  p.src_bf16 = src.dtype == ORDA_BF16;
  p.dst_bf16 = dst.dtype == ORDA_BF16;
  if (p.rows == 1 || (p.lds == p.cols && p.ldd == p.cols)) {
    p.cols *= p.rows;
    p.rows = 1;
  }
  return p;
}

// How the gradients are cut: launches of up to kGradParts of them, pieces of a row,
// one sum for each workgroup.
struct Cut {
  std::vector<GradPart> parts;   // those that have values
  struct Launch {
    size_t from, to;
    int64_t pieces;
    int blocks, first;           // of its sums
  };
  std::vector<Launch> launches;
  int sums = 0;
  int64_t bytes = 0;             // of all gradients
  bool in_place = false;
};

int64_t pieces_of(const GradPart& p) { return p.rows * ceil_div(p.cols, kGradPiece); }

// Workgroups of a launch: eight a CU; and of all together, each of which has a sum that
// every scaling workgroup adds up by itself.
constexpr int64_t kBlocks = 2048, kSums = 4096;

// The memory's cache: gradients beyond it are read past it for the norm (4.29 GB of fp32:
// 612 us, through it 730), smaller ones are read from it by the scaling (42 MB: 12 us,
// had the norm's reads gone past it 16).
constexpr int64_t kCache = int64_t{256} << 20;

void check_count(int64_t count) {
  if (count < 0 || count > kMostGradients) fail(ORDA_ERR_INVALID, "at most 2^20 gradients");
}

Cut cut(const orda_gradient* g, int64_t count, bool scale) {
  check_count(count);
  if (count > 0 && !g) fail(ORDA_ERR_INVALID, "null argument");
  Cut c;
  c.parts.reserve(count);
  int64_t values = 0;
  bool placed[2] = {false, false};
  for (int64_t i = 0; i < count; ++i) {
    const orda_tensor &s = g[i].src, &d = g[i].dst;
    check_view(s, "a gradient");
    to_dtype(s.dtype, "a gradient");
    if (s.location != ORDA_DEVICE) fail(ORDA_ERR_INVALID, "a gradient must be on the device");
    if (s.rows > kMostValues || s.cols > kMostValues || (s.cols > 0 && s.rows > kMostValues / s.cols))
      fail(ORDA_ERR_INVALID, "at most 2^40 values");
    values += s.rows * s.cols;
    if (values > kMostValues) fail(ORDA_ERR_INVALID, "at most 2^40 values");
    if (s.rows == 0 || s.cols == 0) continue;
    placed[d.data != nullptr] = true;
    if (d.data) {
      check_view(d, "a destination");
      to_dtype(d.dtype, "a destination");
      if (d.location != ORDA_DEVICE) fail(ORDA_ERR_INVALID, "a destination must be on the device");
      if (d.rows != s.rows || d.cols != s.cols)
        fail(ORDA_ERR_INVALID, "the destination of gradient %lld must be [%lld, %lld]", static_cast<long long>(i),
             static_cast<long long>(s.rows), static_cast<long long>(s.cols));
    }
    c.bytes += s.rows * s.cols * (s.dtype == ORDA_BF16 ? 2 : 4);
    c.parts.push_back(part_of(s, scale && d.data ? d : s));
  }
  if (scale && placed[0] && placed[1]) fail(ORDA_ERR_INVALID, "either all gradients have a destination or none");
  c.in_place = !placed[1];
  int64_t pieces = 0;
  for (const GradPart& p : c.parts) pieces += pieces_of(p);
  for (size_t at = 0; at < c.parts.size();) {
    Cut::Launch l{at, std::min(at + kGradParts, c.parts.size()), 0, 0, c.sums};
    for (; at < l.to; ++at) {
      c.parts[at].first = l.pieces;
      l.pieces += pieces_of(c.parts[at]);
    }
    // its share of 2048, or as many as have eight pieces each: with the share alone 110
    // gradients of 1.05 GB, two launches, took 226 us for the norm, so 212
    const int64_t share = kBlocks * l.pieces / pieces, most = kSums * l.pieces / pieces;
    l.blocks = static_cast<int>(std::max<int64_t>(1, std::min({l.pieces, std::max(share, std::min(kBlocks, l.pieces / 8)), most})));
    c.sums += l.blocks;
    c.launches.push_back(l);
  }
  return c;
}

// Memory from `from` to `to`, rows of `cols` bytes `ld` bytes apart.
struct Span {
  uintptr_t from, to;
  int64_t cols, ld;
  bool written;
  bool operator<(const Span& o) const { return from < o.from; }
};
bool meet(const Span& a, const Span& b) {
  if (a.to <= b.from || b.to <= a.from) return false;
  // column ranges of one frame
  const int64_t ld = a.ld;
  if (ld == b.ld && a.cols < ld && b.cols < ld) {
    const int64_t d = static_cast<int64_t>(b.from - a.from) % ld;   // (from is sorted)
    return !(d >= a.cols && d + b.cols <= ld);
  }
  return true;
}
void check_apart(const Cut& c) {
  std::vector<Span> spans;
  spans.reserve(2 * c.parts.size());
  auto add = [&](const void* p, const GradPart& g, int64_t ld, int64_t es, bool written) {
    const auto from = reinterpret_cast<uintptr_t>(p);
    spans.push_back({from, from + ((g.rows - 1) * ld + g.cols) * es, g.cols * es, g.rows == 1 ? 0 : ld * es, written});
  };
  for (const GradPart& g : c.parts) {
    add(g.src, g, g.lds, g.src_bf16 ? 2 : 4, c.in_place);
    if (!c.in_place) add(g.dst, g, g.ldd, g.dst_bf16 ? 2 : 4, true);
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 0; i < spans.size(); ++i)
    for (size_t j = i + 1; j < spans.size() && spans[j].from < spans[i].to; ++j)
      if ((spans[i].written || spans[j].written) && meet(spans[i], spans[j]))
        fail(ORDA_ERR_INVALID, "gradients that are written share memory with others");
}

// Every launch has its share of the workgroups, and one at least.
int64_t sum_bytes(int64_t count) {
  const int64_t launches = ceil_div(count, kGradParts);
  return count == 0 ? 0 : ((std::min(launches * kBlocks, kSums) + launches) * 8 + 255) / 256 * 256;
}

void run(int32_t device, hipStream_t st, const Cut& c, int64_t count, bool scale, double max_norm, double eps, float* norm, void* ws,
         int64_t ws_bytes) {
  const int64_t need = sum_bytes(count);
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0) fail(ORDA_ERR_INVALID, "workspace must be 256-byte aligned");
  if (ws_bytes < need || (need > 0 && !ws))
    fail(ORDA_ERR_INVALID, "workspace of %lld bytes, %lld needed", static_cast<long long>(ws_bytes),
         static_cast<long long>(need));
  const DeviceScope scope(device);
  auto* sums = static_cast<double*>(ws);
  auto args = [&](const Cut::Launch& l) {
    GradArgs a{};
    std::copy(c.parts.begin() + l.from, c.parts.begin() + l.to, a.part);
    a.count = static_cast<int32_t>(l.to - l.from);
    a.pieces = l.pieces;
    a.sums = sums + l.first;
    return a;
  };
  for (const Cut::Launch& l : c.launches) hip_check(launch_grad_sums(args(l), l.blocks, c.bytes > kCache, st), "gradient norm");
  if (!scale || c.launches.empty()) {
    hip_check(launch_grad_norm(sums, c.sums, norm, st), "gradient norm");
    return;
  }
  for (size_t i = 0; i < c.launches.size(); ++i) {
    GradArgs a = args(c.launches[i]);
    a.all = sums;
    a.n_sums = c.sums;
    a.in_place = c.in_place;
    a.max_norm = max_norm;
    a.eps = eps;
    a.norm = i == 0 ? norm : nullptr;
    hip_check(launch_grad_scale(a, c.launches[i].blocks, st), "gradient clipping");
  }
}

}  // namespace
}  // namespace orda

using namespace orda;

extern "C" {

int32_t orda_clip_gradients_workspace(int64_t count, int64_t* bytes, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!bytes) fail(ORDA_ERR_INVALID, "null argument");
    check_count(count);
    *bytes = sum_bytes(count);
  });
}

int32_t orda_gradient_norm(int32_t device, void* hip_stream, const orda_gradient* gradients, int64_t count, float* norm,
                           void* workspace, int64_t workspace_bytes, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!norm) fail(ORDA_ERR_INVALID, "null argument");
    const Cut c = cut(gradients, count, false);
    run(device, static_cast<hipStream_t>(hip_stream), c, count, false, 0., 0., norm, workspace, workspace_bytes);
  });
}

int32_t orda_clip_gradients(int32_t device, void* hip_stream, const orda_gradient* gradients, int64_t count,
                            double max_norm, double eps, float* norm, void* workspace, int64_t workspace_bytes, char* err,
                            size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!norm) fail(ORDA_ERR_INVALID, "null argument");
    if (!(max_norm >= 0.)) fail(ORDA_ERR_INVALID, "max_norm must be >= 0");
    if (!(eps >= 0.) || !isfinite(eps)) fail(ORDA_ERR_INVALID, "eps must be >= 0 and finite");
    const Cut c = cut(gradients, count, true);
    check_apart(c);
    run(device, static_cast<hipStream_t>(hip_stream), c, count, true, max_norm, eps, norm, workspace, workspace_bytes);
  });
}

}  // extern "C"
