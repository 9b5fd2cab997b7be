// linear_ce.cpp — the linear cross entropy that keeps no logits
// (orda_linear_ce_* of include/orda/orda.h): the rows that have a label are
// compacted, and each piece of the vocabulary's columns is one product whose
// epilogue leaves row statistics (forward) or the gradient of the logits
// (backward, followed by the products of grad_hidden and grad_weight). The
// count of those rows stays on the device, the scratch is the caller's: the
// calls queue their kernels and return, and can be captured into a graph.
#include <algorithm>

#include "orda_host.h"

namespace orda {
namespace {

// A product's operand is read with 32-bit byte offsets inside a tile of 256 rows:
// 255 rows of 2^21 columns in three planes of bf16 are 3.2 GB. A row of an operand
// is a row of hidden or weight, a column of hidden (its transpose) or a piece's
// gradient of the logits.
constexpr int64_t kMaxWidth = int64_t{1} << 20, kMaxRows = int64_t{1} << 21, kMaxPiece = int64_t{1} << 21;
constexpr int64_t kMaxColumns = int64_t{1} << 30;
// Scratch a piece may take: the larger the piece, the fewer the passes that
// read and write the fp32 grad_hidden.
constexpr int64_t kPieceBytes = int64_t{1} << 30;

struct Ce {
  DType t;
  int64_t n, h, v;
  const void *x, *w;
  int64_t ldx, ldw;
  bool planes;       // fp32: every product over three-plane operands
  bool direct;       // small fp32 calls: the logits in memory, fp32 operands
  bool few;          // few rows (bf16, or direct): the logits by waves of 16 classes
  bool stage_w;      // weights that the products cannot read in place
  bool gh, gw;       // backward: the gradients asked for
  bool backward;
  int64_t hp;        // pitch of the compact hidden rows, plane width with planes
  int64_t piece;     // columns of a piece
};

int64_t ds_pitch(const Ce& c, int64_t cols) { return c.planes ? 3 * round64(cols) : logits_pitch(cols, DType::BF16); }

// Weights that the products cannot read in place (few rows' logits can).
bool copies_weight(const Ce& c) { return c.stage_w && (!c.few || c.gh); }

int64_t column_bytes(const Ce& c) {   // of scratch, for each column of a piece
  int64_t b = c.planes ? 6 * c.hp : copies_weight(c) ? dtype_size(c.t) * c.hp : 0;
  b += c.backward ? round64(c.n) * (c.planes ? 6 : 2) : c.few ? (c.n * 16 + 63) / 64 : (c.n * 16 + 255) / 256;
  return b;
}

int64_t stat_tiles(const Ce& c, int64_t cols) {
  return c.few ? ce_few_tiles(cols) : c.direct ? ce_direct_tiles(cols) : gemm_stat_tiles(cols);
}

void choose_direct(Ce& c, bool one_piece);
int64_t scratch_bytes(const Ce& c);

// us of the logits of few rows by waves of 16 classes: the weight's bytes at the rate
// that the rows' way from the caches leaves, or a wave's own way through K. fp32
// (beside fp32 tiles): 32000 x 4096, one row 117 (531), 64 rows 333 (546); 8000 x
// 1024, 64 rows 49 (31, taken).
double few_us(const Ce& c) {
  const bool f32 = c.t == DType::F32;
  const double terms = static_cast<double>(c.v) * static_cast<double>(c.h) * (f32 ? 2.0 : 1.0);
  const double all = terms * (c.n <= 16 ? 4.5e-7 : c.n <= 32 ? 6.9e-7 : 11.8e-7) + 2.0;
  const double f = c.n <= 16 ? 1.0 : c.n <= 32 ? 2.0 : 4.0;
  const double wave = static_cast<double>(c.h) * (f32 ? (0.5 + 0.62 * f) / 64 : (0.35 + 0.5 * f) / 128);
  return std::max(all, wave);
}

// Whether bf16 logits of few rows go that way: where it is quicker than tiles of
// 256, each of which takes as long as K asks while fewer tiles than CUs leave the
// memory idle. Both sides' us: 14334 x 4032, 18 rows 31 against 75; 32000 x 2048, one
// row 23 against 41, 32 rows 47 against 40; 2000 x 4096, 16 rows 31 against 70, 64
// rows 74 against 70; 131072 x 4096, one row 200 against 184 (all tiles' CUs at work:
// the weight at 5.8 TB/s). Weights that the tiles cannot read in place take a copy
// first, 5.9 TB/s.
bool few_rows(const Ce& c) {
  if (c.planes || c.n > kCeFewRows) return false;
  const double terms = static_cast<double>(c.v) * static_cast<double>(c.hp);
  const double rounds = static_cast<double>(((c.v + 255) / 256 + 255) / 256);
  const double tiles = std::max(rounds * (static_cast<double>(c.hp) * 0.0155 + 8.0), terms * 2 / 5.8e6);
  return few_us(c) < tiles + (c.stage_w && !c.gh ? terms * 4 / 5.9e6 : 0.0);
}

Ce make_ce(const orda_linear_ce& a, int64_t labels, bool backward, bool gh, bool gw) {
  check_view(a.hidden, "hidden");
  check_view(a.weight, "weight");
  Ce c{};
  c.t = to_dtype(a.hidden.dtype, "hidden");
  if (to_dtype(a.weight.dtype, "weight") != c.t) fail(ORDA_ERR_INVALID, "hidden and weight must share one dtype");
  if (a.hidden.location != ORDA_DEVICE || a.weight.location != ORDA_DEVICE)
    fail(ORDA_ERR_INVALID, "hidden and weight must be on the device");
  c.n = a.hidden.rows;
  c.h = a.hidden.cols;
  c.v = a.weight.rows;
  if (a.weight.cols != c.h)
    fail(ORDA_ERR_INVALID, "weight has %lld columns, hidden %lld", static_cast<long long>(a.weight.cols),
         static_cast<long long>(c.h));
  if (labels != c.n)
    fail(ORDA_ERR_INVALID, "%lld labels for %lld rows", static_cast<long long>(labels), static_cast<long long>(c.n));
  if (c.h < 1 || c.v < 1) fail(ORDA_ERR_INVALID, "hidden width and vocabulary must be > 0");
  if (c.h > kMaxWidth || c.n > kMaxRows || c.v > kMaxColumns)
    fail(ORDA_ERR_INVALID, "at most 2^20 columns, 2^21 rows and 2^30 classes");
  if (!(a.label_smoothing >= 0.f && a.label_smoothing <= 1.f))
    fail(ORDA_ERR_INVALID, "label_smoothing must be in [0, 1]");
  if (a.vocab_piece < 0) fail(ORDA_ERR_INVALID, "vocab_piece must be >= 0");
  c.x = a.hidden.data;
  c.w = a.weight.data;
  c.ldx = tensor_ld(a.hidden);
  c.ldw = tensor_ld(a.weight);
  c.planes = c.t == DType::F32;
  c.stage_w = !(c.ldw <= kMaxWidth && c.ldw % 8 == 0 && c.h % 8 == 0 && reinterpret_cast<uintptr_t>(c.w) % 16 == 0);
  c.hp = c.planes ? round64(c.h) : round8(c.h);
  c.backward = backward;
  c.gh = gh;
  c.gw = gw;
  c.few = few_rows(c);
  // Pieces of whole column tiles, all but the last alike.
  int64_t most = a.vocab_piece > 0 ? a.vocab_piece : std::max<int64_t>(kPieceBytes / std::max<int64_t>(column_bytes(c), 1), 4096);
  // (a logits product's tiles, of 128 rows at least, in one launch)
  most = std::min({most, kMaxPiece, most_blocks(256) / std::max<int64_t>((c.n + 127) / 128, 1) * 256});
  most = std::max<int64_t>(most / 256 * 256, 256);
  const int64_t pieces = (c.v + most - 1) / most;
  c.piece = pieces == 1 ? c.v : ((c.v + pieces - 1) / pieces + 255) / 256 * 256;
  // (The planes' scratch cuts pieces that the direct form, which makes no planes, does not need.)
  choose_direct(c, c.v <= (a.vocab_piece > 0 ? c.piece : kMaxPiece));
  return c;
}

// The scratch of a call, laid out from base.
struct Scratch {
  CeRows rows;
  void* x;           // compact hidden rows, or their planes
  void* xt;          // transposed: grad_weight's K-major operand
  void* w;           // a piece of the weights, padded or as planes
  void* ds;          // gradient of a piece's logits
  float* gh;         // grad_hidden of the compact rows
  float* logits;     // direct: the logits; the gradient of the logits is ds
  float4 *stats, *state, *coef;
  float* xy;
  float* split;
  int64_t split_bytes, bytes;
};

GemmArgs product(const Ce& c, const Scratch& s) {
  GemmArgs g{};
  g.nprob = 1;
  g.in_type = DType::BF16;
  g.a_kmajor = true;
  g.alpha = 1.f;
  g.dyn_rows = s.rows.count;
  g.split_ws = s.split;
  g.split_ws_bytes = s.split_bytes;
  return g;
}

// The piece's logits product: columns [v0, v0 + cols).
GemmArgs logits_product(const Ce& c, const Scratch& s, int64_t v0, int64_t cols) {
  GemmArgs g = product(c, s);
  g.M = c.n;
  g.N = cols;
  g.K = c.hp;
  g.lda = c.hp;
  g.ldb = c.stage_w ? c.hp : c.ldw;
  g.prob[0] = {s.x, c.stage_w ? s.w : static_cast<const char*>(c.w) + v0 * c.ldw * 2, nullptr};
  g.b_kmajor = true;
  g.group_m = 8;
  g.ce.labels = s.rows.labels;
  g.ce.col0 = v0;
  if (c.planes) {
    g.lda = g.ldb = 3 * c.hp;
    g.plane_a = g.plane_b = c.hp;
    g.prob[0] = {s.x, s.w, nullptr};
  } else {
    g.K = c.h;
  }
  return g;
}

// The piece's share of grad_hidden: added to the pieces before it in s.gh, and
// with the last piece written to its rows' places.
GemmArgs grad_hidden_product(const Ce& c, const Scratch& s, const orda_tensor* gh, int64_t v0, int64_t cols) {
  GemmArgs g = product(c, s);
  g.M = c.n;
  g.N = c.h;
  g.K = c.planes ? round64(cols) : cols;
  g.lda = ds_pitch(c, c.piece);
  g.ldb = c.stage_w ? c.hp : c.ldw;
  g.ldc = round8(c.h);
  g.epi = GemmEpilogue::StoreF32;
  g.group_m = 4;
  g.share_rounds = true;
  g.ce.accum = v0 > 0;
  if (gh != nullptr && v0 + cols == c.v) {
    g.ce.src = s.rows.src;
    g.ce.out = gh->data;
    g.ce.ldo = tensor_ld(*gh);
    g.ce.out_type = c.t;
  }
  g.prob[0] = {s.ds, c.stage_w ? s.w : static_cast<const char*>(c.w) + v0 * c.ldw * 2, s.gh};
  if (c.planes) {
    g.ldb = 3 * c.hp;
    g.plane_a = round64(c.piece);
    g.plane_b = c.hp;
    g.prob[0].b = s.w;
  }
  return g;
}

GemmArgs grad_weight_product(const Ce& c, const Scratch& s, void* gw, int64_t ldg, int64_t v0, int64_t cols) {
  GemmArgs g = product(c, s);
  g.M = c.h;
  g.N = cols;
  g.K = c.planes ? round64(c.n) : c.n;
  g.lda = round64(c.n);
  g.ldb = ds_pitch(c, c.piece);
  g.ldc = ldg;
  g.c_trans = true;
  g.c_type = c.t;
  g.epi = GemmEpilogue::StoreF32;
  g.group_m = 8;
  g.prob[0] = {s.xt, s.ds, static_cast<char*>(gw) + v0 * ldg * dtype_size(c.t)};
  if (c.planes) {
    g.lda = 3 * round64(c.n);
    g.plane_a = round64(c.n);
    g.plane_b = round64(c.piece);
  }
  return g;
}

// The same of few rows, the weights read where they are.
CeFewArgs few_logits(const Ce& c, const Scratch& s, int64_t v0, int64_t cols) {
  CeFewArgs f{};
  f.x = s.x;
  f.ldx = c.hp;
  f.w = static_cast<const char*>(c.w) + v0 * c.ldw * dtype_size(c.t);
  f.ldw = c.ldw;
  f.n = c.n;
  f.k = c.h;
  f.cols = cols;
  f.col0 = v0;
  f.rows = s.rows;
  f.xy = s.xy;
  f.coef = s.coef;
  f.stats = s.stats;
  f.stats_ld = stat_tiles(c, c.piece);
  f.ds = s.ds;
  return f;
}

// The direct form's products: fp32 operands, rows from the count on zeros.
int64_t direct_pitch(const Ce& c) { return logits_pitch(c.v, DType::F32); }
GemmArgs direct_product(const Ce& c, const Scratch& s) {
  GemmArgs g{};
  g.nprob = 1;
  g.in_type = DType::F32;
  g.a_kmajor = true;
  g.alpha = 1.f;
  g.epi = GemmEpilogue::StoreF32;
  g.split_ws = s.split;
  g.split_ws_bytes = s.split_bytes;
  return g;
}
const void* direct_weight(const Ce& c, const Scratch& s) { return c.stage_w ? s.w : c.w; }
GemmArgs direct_logits_product(const Ce& c, const Scratch& s) {
  GemmArgs g = direct_product(c, s);
  g.M = c.n;
  g.N = c.v;
  g.K = c.h;
  g.lda = c.hp;
  g.ldb = c.stage_w ? c.hp : c.ldw;
  g.ldc = direct_pitch(c);
  g.b_kmajor = true;
  g.group_m = 8;
  g.prob[0] = {s.x, direct_weight(c, s), s.logits};
  return g;
}
GemmArgs direct_hidden_product(const Ce& c, const Scratch& s) {
  GemmArgs g = direct_product(c, s);
  g.M = c.n;
  g.N = c.h;
  g.K = c.v;
  g.lda = direct_pitch(c);
  g.ldb = c.stage_w ? c.hp : c.ldw;
  g.ldc = round8(c.h);
  g.group_m = 4;
  g.share_rounds = true;
  g.prob[0] = {s.ds, direct_weight(c, s), s.gh};
  return g;
}
GemmArgs direct_weight_product(const Ce& c, const Scratch& s, void* gw, int64_t ldg) {
  GemmArgs g = direct_product(c, s);
  g.M = c.h;
  g.N = c.v;
  g.K = c.n;
  g.lda = round64(c.n);
  g.ldb = direct_pitch(c);
  g.ldc = ldg;
  g.c_trans = true;
  g.group_m = 8;
  g.prob[0] = {s.xt, s.ds, gw};
  return g;
}

// Whether an fp32 call keeps its logits and multiplies fp32 operands: where the
// passes that make planes of the weights, and tiles of 256 rows, cost more than
// the logits' way through memory. Both sides by the products' own measure
// (gemm_us; 4.2 us for every 32 elements of K and 20 us a round of 256 tiles over
// planes) and 4 TB/s: 256 x 512 x 8192, forward and backward, 250 us of kernels
// over planes. It takes the vocabulary in one piece (one_piece: the caller allows
// that), and where the planes would be cut by their scratch, it stays within the
// same bound itself: the losses of one row at 131072 x 4096 take 1 MB and 0.45 ms (the
// planes 770 MB and 2.45), of 64 rows 1.21 ms (2.47), both gradients too 2.1 (4.1) and
// 3.2 (4.4).
void choose_direct(Ce& c, bool one_piece) {
  if (!c.planes || !one_piece || c.n > 8192) return;
  const double pass = (static_cast<double>(c.v) + c.n) * c.h * 10 * 0.25e-6;
  auto tiles = [](int64_t m, int64_t n) { return (m + 255) / 256 * ((n + 255) / 256); };
  auto rounds = [](int64_t t, int64_t k) { return static_cast<double>((t + 255) / 256) * (k / 32.0 * 4.2 + 20.0); };
  double planes = pass + rounds(tiles(c.n, c.v), c.hp);
  Ce d = c;
  d.planes = false;
  d.hp = round8(c.h);
  const Scratch none{};
  double logits = gemm_us(direct_logits_product(d, none)) + static_cast<double>(c.n) * c.v * 8 * 0.25e-6 + 4.0;
  d.few = c.n <= kCeFewRows && few_us(d) < logits;
  if (d.few) logits = few_us(d);
  double direct = logits;
  if (c.stage_w && (!d.few || c.gh)) direct += static_cast<double>(c.v) * c.h * 8 * 0.25e-6;
  if (c.backward) {
    const double kv = static_cast<double>(c.v);
    // over planes K is split until the chip is full
    if (c.gh) planes += std::max(tiles(c.n, c.h) * kv / 32 * 4.2 / 256, 20.0) + 12.0;
    if (c.gw) planes += std::max(tiles(c.h, c.v) / 256.0, 1.0) * (round64(c.n) / 32.0 * 4.2 + 12.0);
    if (c.gh) direct += gemm_us(direct_hidden_product(d, none)) + 4.0;
    if (c.gw) direct += gemm_us(direct_weight_product(d, none, nullptr, c.h));
    if (!d.few) direct += static_cast<double>(c.n) * c.v * 8 * 0.25e-6;
  }
  if (direct >= planes) return;
  d.direct = true;
  const bool cut = c.piece < c.v;
  d.piece = d.v;
  if (!cut || scratch_bytes(d) <= kPieceBytes) c = d;
}

// (Sizes depend on which pointers are set, so a layout is made from a base that
// is not null also where only its size counts.)
Scratch lay_out(const Ce& c, void* base) {
  Scratch s{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) -> void* {
    char* p = static_cast<char*>(base) + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const int64_t np = round64(c.n);
  s.rows.count = static_cast<int64_t*>(take(8));
  s.rows.src = static_cast<int32_t*>(take(c.n * 4));
  s.rows.pos = static_cast<int32_t*>(take(c.n * 4));
  s.rows.labels = static_cast<int64_t*>(take(c.n * 8));
  s.x = take(np * c.hp * (c.planes ? 6 : dtype_size(c.t)));
  if (c.direct) {
    const int64_t ld = direct_pitch(c);
    if (copies_weight(c)) s.w = take(c.v * c.hp * 4);
    if (!c.few) {
      s.logits = static_cast<float*>(take(c.n * ld * 4));
      s.split_bytes = gemm_split_bytes(direct_logits_product(c, s));
    }
    if (!c.backward) {
      s.stats = static_cast<float4*>(take(c.n * stat_tiles(c, c.v) * 16));
      s.xy = static_cast<float*>(take(c.n * 4));
    } else {
      s.coef = static_cast<float4*>(take(c.n * 16));
      s.ds = take(c.n * ld * 4);
      if (c.gh) {
        s.gh = static_cast<float*>(take(c.n * round8(c.h) * 4));
        s.split_bytes = std::max(s.split_bytes, gemm_split_bytes(direct_hidden_product(c, s)));
      }
      if (c.gw) {
        s.xt = take(c.h * np * 4);
        s.split_bytes = std::max(s.split_bytes, gemm_split_bytes(direct_weight_product(c, s, nullptr, c.h)));
      }
    }
    s.split = s.split_bytes > 0 ? static_cast<float*>(take(s.split_bytes)) : nullptr;
    s.bytes = at;
    return s;
  }
  if (c.planes) s.w = take(round64(c.piece) * 6 * c.hp);
  else if (copies_weight(c)) s.w = take(c.piece * c.hp * 2);
  if (!c.backward) {
    const int64_t tiles = stat_tiles(c, c.piece);
    s.stats = static_cast<float4*>(take(c.n * tiles * 16));
    s.state = static_cast<float4*>(c.piece < c.v ? take(c.n * 16) : nullptr);
    s.xy = static_cast<float*>(take(c.n * 4));
  } else {
    s.coef = static_cast<float4*>(take(c.n * 16));
    s.ds = take(np * ds_pitch(c, c.piece) * 2);
    if (c.gh && c.piece < c.v) s.gh = static_cast<float*>(take(c.n * round8(c.h) * 4));
    if (c.gw) s.xt = take(c.h * np * (c.planes ? 6 : 2));
    // a piece and the last one split differently
    const int64_t last = c.v - (c.v - 1) / c.piece * c.piece;
    for (const int64_t cols : {c.piece, last}) {
      if (c.gh) s.split_bytes = std::max(s.split_bytes, gemm_split_bytes(grad_hidden_product(c, s, nullptr, 0, cols)));
      if (c.gw) s.split_bytes = std::max(s.split_bytes, gemm_split_bytes(grad_weight_product(c, s, nullptr, c.h, 0, cols)));
    }
    s.split = s.split_bytes > 0 ? static_cast<float*>(take(s.split_bytes)) : nullptr;
  }
  s.bytes = at;
  return s;
}

int64_t scratch_bytes(const Ce& c) { return lay_out(c, reinterpret_cast<void*>(uintptr_t{256})).bytes; }

Scratch check_scratch(const Ce& c, void* workspace, int64_t bytes) {
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) fail(ORDA_ERR_INVALID, "workspace must be 256-byte aligned");
  if (!workspace) fail(ORDA_ERR_INVALID, "null workspace");
  const Scratch s = lay_out(c, workspace);
  if (bytes < s.bytes)
    fail(ORDA_ERR_INVALID, "workspace of %lld bytes, %lld needed", static_cast<long long>(bytes),
         static_cast<long long>(s.bytes));
  return s;
}

CePrepArgs prepare_rows(const orda_linear_ce& a, const Ce& c, const Scratch& s) {
  CePrepArgs p{};
  p.x = c.x;
  p.ldx = c.ldx;
  p.n = c.n;
  p.h = c.h;
  p.labels = a.labels;
  p.v = c.v;
  p.ignore = a.ignore_index;
  p.rows = s.rows;
  p.dst = s.x;
  p.pitch = c.hp;
  p.whole = c.direct;
  return p;
}

// The piece's weights where the products do not read them in place.
void stage_weights(const Ce& c, const Scratch& s, int64_t v0, int64_t cols, hipStream_t st) {
  if (c.planes)
    hip_check(launch_split3_rows(static_cast<const float*>(c.w) + v0 * c.ldw, c.ldw, cols, c.h, s.w, round64(cols),
                                 c.hp, st),
              "linear cross entropy weights");
  else if (copies_weight(c))
    hip_check(launch_ce_stage(DType::BF16, static_cast<const char*>(c.w) + v0 * c.ldw * 2, c.ldw, s.w, c.hp, cols, c.h,
                              st),
              "linear cross entropy weights");
}

void stage_direct(const Ce& c, const Scratch& s, hipStream_t st) {
  if (copies_weight(c))
    hip_check(launch_ce_stage(DType::F32, c.w, c.ldw, s.w, c.hp, c.v, c.h, st), "linear cross entropy weights");
}

// The direct form's logits, the parts of a split product left apart.
CeDirectArgs direct_logits(const Ce& c, const Scratch& s, hipStream_t st) {
  GemmArgs g = direct_logits_product(c, s);
  const GemmSplit plan = gemm_split_plan(g);
  g.partials_only = plan.splits > 1;
  hip_check(launch_gemm(g, st), "linear cross entropy logits");
  CeDirectArgs d{};
  d.rows = s.rows;
  d.v = c.v;
  d.logits = plan.splits > 1 ? s.split : s.logits;
  d.ld = plan.splits > 1 ? plan.ldp : g.ldc;
  d.stride = plan.splits > 1 ? plan.stride : 0;
  d.splits = plan.splits > 1 ? plan.splits : 1;
  d.stats = s.stats;
  d.stats_ld = stat_tiles(c, c.v);
  d.xy = s.xy;
  d.coef = s.coef;
  d.grad = static_cast<float*>(s.ds);
  d.grad_ld = g.ldc;
  return d;
}

CeLossArgs losses(const orda_linear_ce& a, const Ce& c, const Scratch& s, float* nll, float* lse) {
  CeLossArgs l{};
  l.rows = s.rows;
  l.stats = s.stats;
  l.state = s.state;
  l.first = l.last = true;
  l.xy = s.xy;
  l.smooth_each = a.label_smoothing / static_cast<float>(c.v);
  l.target = 1.f - a.label_smoothing;
  l.nll = nll;
  l.lse = lse;
  return l;
}

void forward(const orda_linear_ce& a, const Ce& c, const Scratch& s, float* nll, float* lse, hipStream_t st) {
  CePrepArgs p = prepare_rows(a, c, s);
  p.nll = nll;
  p.lse_out = lse;
  hip_check(launch_ce_prep(p, c.t, c.planes, st), "linear cross entropy rows");
  if (c.direct) {
    stage_direct(c, s, st);
    if (c.few) hip_check(launch_ce_few(few_logits(c, s, 0, c.v), c.t, false, st), "linear cross entropy logits");
    else hip_check(launch_ce_direct(direct_logits(c, s, st), c.n, false, st), "linear cross entropy losses");
    CeLossArgs l = losses(a, c, s, nll, lse);
    l.stats_ld = l.tiles = stat_tiles(c, c.v);
    hip_check(launch_ce_losses(l, c.n, st), "linear cross entropy losses");
    return;
  }
  for (int64_t v0 = 0; v0 < c.v; v0 += c.piece) {
    const int64_t cols = std::min(c.piece, c.v - v0);
    stage_weights(c, s, v0, cols, st);
    const int64_t stats_ld = stat_tiles(c, c.piece);
    if (c.few) {
      hip_check(launch_ce_few(few_logits(c, s, v0, cols), c.t, false, st), "linear cross entropy logits");
    } else {
      GemmArgs g = logits_product(c, s, v0, cols);
      g.epi = GemmEpilogue::CeStats;
      g.ce.stats = s.stats;
      g.ce.stats_ld = stats_ld;
      g.ce.xy = s.xy;
      hip_check(launch_gemm(g, st), "linear cross entropy logits");
    }
    CeLossArgs l = losses(a, c, s, nll, lse);
    l.stats_ld = stats_ld;
    l.tiles = stat_tiles(c, cols);
    l.first = v0 == 0;
    l.last = v0 + cols == c.v;
    hip_check(launch_ce_losses(l, c.n, st), "linear cross entropy losses");
  }
}

void backward(const orda_linear_ce& a, const Ce& c, const Scratch& s, const CeGradRows& gr, orda_tensor* gh, orda_tensor* gw,
              hipStream_t st) {
  CePrepArgs p = prepare_rows(a, c, s);
  p.grad = gr;
  p.grad.smooth_each = a.label_smoothing / static_cast<float>(c.v);
  p.grad.target = 1.f - a.label_smoothing;
  p.grad.coef = s.coef;
  p.trans = s.xt;
  p.ldt = round64(c.n);
  if (c.gh) {
    p.zero = gh->data;
    p.ldz = tensor_ld(*gh);
  }
  hip_check(launch_ce_prep(p, c.t, c.planes, st), "linear cross entropy rows");
  if (c.direct) {
    stage_direct(c, s, st);
    if (c.few) {
      CeFewArgs f = few_logits(c, s, 0, c.v);
      f.ldds = direct_pitch(c);
      hip_check(launch_ce_few(f, c.t, true, st), "linear cross entropy gradient");
    } else {
      hip_check(launch_ce_direct(direct_logits(c, s, st), c.n, true, st), "linear cross entropy gradient");
    }
    if (c.gh) {
      hip_check(launch_gemm(direct_hidden_product(c, s), st), "grad_hidden");
      hip_check(launch_ce_scatter(s.gh, round8(c.h), s.rows, c.n, c.h, static_cast<float*>(gh->data), tensor_ld(*gh), st),
                "grad_hidden");
    }
    if (c.gw) hip_check(launch_gemm(direct_weight_product(c, s, gw->data, tensor_ld(*gw)), st), "grad_weight");
    return;
  }
  for (int64_t v0 = 0; v0 < c.v; v0 += c.piece) {
    const int64_t cols = std::min(c.piece, c.v - v0);
    stage_weights(c, s, v0, cols, st);
    if (c.few) {
      CeFewArgs f = few_logits(c, s, v0, cols);
      f.ldds = ds_pitch(c, c.piece);
      hip_check(launch_ce_few(f, c.t, true, st), "linear cross entropy gradient");
    } else {
      GemmArgs g = logits_product(c, s, v0, cols);
      g.epi = GemmEpilogue::CeGrad;
      g.logits_type = DType::BF16;
      g.prob[0].c = s.ds;
      g.ldc = ds_pitch(c, c.piece);
      g.ce.plane = round64(c.piece);
      g.ce.coef = s.coef;
      hip_check(launch_gemm(g, st), "linear cross entropy gradient");
    }
    if (c.gh) hip_check(launch_gemm(grad_hidden_product(c, s, gh, v0, cols), st), "grad_hidden");
    if (c.gw) hip_check(launch_gemm(grad_weight_product(c, s, gw->data, tensor_ld(*gw), v0, cols), st), "grad_weight");
  }
}

bool wanted(const orda_tensor* g) { return g != nullptr && g->data != nullptr; }

void check_grad(const orda_tensor& g, DType t, int64_t rows, int64_t cols, const char* what) {
  check_view(g, what);
  if (to_dtype(g.dtype, what) != t) fail(ORDA_ERR_INVALID, "%s must have its input's dtype", what);
  if (g.location != ORDA_DEVICE) fail(ORDA_ERR_INVALID, "%s must be on the device", what);
  if (g.rows != rows || g.cols != cols)
    fail(ORDA_ERR_INVALID, "%s must be [%lld, %lld]", what, static_cast<long long>(rows), static_cast<long long>(cols));
}

}  // namespace
}  // namespace orda

using namespace orda;

extern "C" {

int32_t orda_linear_ce_workspace(const orda_linear_ce* args, int32_t backward, int64_t* bytes, char* err,
                                 size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!args || !bytes) fail(ORDA_ERR_INVALID, "null argument");
    const Ce c = make_ce(*args, args->n_labels, backward != 0, (backward & 1) != 0, (backward & 2) != 0);
    *bytes = c.n > 0 ? scratch_bytes(c) : 0;
  });
}

int32_t orda_linear_ce_forward(int32_t device, void* hip_stream, const orda_linear_ce* args, float* nll, float* lse,
                               void* workspace, int64_t workspace_bytes, char* err, size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!args) fail(ORDA_ERR_INVALID, "null argument");
    const Ce c = make_ce(*args, args->n_labels, false, false, false);
    if (c.n == 0) return;
    if (!args->labels || !nll || !lse) fail(ORDA_ERR_INVALID, "null argument");
    const Scratch s = check_scratch(c, workspace, workspace_bytes);
    const DeviceScope scope(device);
    forward(*args, c, s, nll, lse, static_cast<hipStream_t>(hip_stream));
  });
}

int32_t orda_linear_ce_backward(int32_t device, void* hip_stream, const orda_linear_ce* args, const float* lse,
                                const float* grad_nll, const float* grad_lse, orda_tensor* grad_hidden,
                                orda_tensor* grad_weight, void* workspace, int64_t workspace_bytes, char* err,
                                size_t err_len) {
  return guarded(err, err_len, [&] {
    if (!args) fail(ORDA_ERR_INVALID, "null argument");
    const Ce c = make_ce(*args, args->n_labels, true, wanted(grad_hidden), wanted(grad_weight));
    if (c.gh) check_grad(*grad_hidden, c.t, c.n, c.h, "grad_hidden");
    if (c.gw) check_grad(*grad_weight, c.t, c.v, c.h, "grad_weight");
    if (!c.gh && !c.gw) return;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (c.n == 0) {   // no rows: a weight gradient of zeros
      if (!c.gw) return;
      const DeviceScope scope(device);
      hip_check(launch_zero_rows(c.t, grad_weight->data, tensor_ld(*grad_weight), c.v, c.h, st), "grad_weight");
      return;
    }
    if (!args->labels || !lse) fail(ORDA_ERR_INVALID, "null argument");
    const Scratch s = check_scratch(c, workspace, workspace_bytes);
    const DeviceScope scope(device);
    CeGradRows gr{};
    gr.lse = lse;
    gr.grad_nll = grad_nll;
    gr.grad_lse = grad_lse;
    backward(*args, c, s, gr, grad_hidden, grad_weight, st);
  });
}

}  // extern "C"
