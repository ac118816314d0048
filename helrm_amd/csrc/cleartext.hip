// cleartext.hip -- C ABI of the operators that train and score in the clear:
// argument checks, the division of a workspace, and the order of the launches.
#include <algorithm>
#include <climits>
#include "cleartext.h"
#include "embedding.h"
#include "norm.h"
#include "preference.h"
#include "products.h"
#include "skinny.h"
#include "teacher.h"
#include "../../include/helrm_hip.h"

namespace {

using clr::require;

// Hands out pieces of a workspace, or only counts where there is none.
struct Arena {
  char* base;
  size_t used = 0;
  template <class T> T* take(size_t n) {
    const size_t at = used;
    used += clr::align256(n * sizeof(T));
    return base ? (T*)(base + at) : nullptr;
  }
  void* bytes(size_t n) { return take<char>(n); }
};

void check_type(int t) { require(t == DT_F32 || t == DT_BF16 || t == DT_F16, "unknown element type"); }
void check_space(const void* ws, size_t have, size_t need) {
  require(have >= need && (ws || !need), "workspace too small");
  require((uintptr_t)ws % 256 == 0, "workspace not aligned to 256 bytes");
}
// A matrix is there, and a row's stride covers it.
void check_matrix(const void* p, long ld, long rows, long width, const char* what) {
  require(p || !rows, what);
  require(rows <= 1 || ld >= width, what);
}
constexpr long MAX_ROWS = 1L << 30;
constexpr long MAX_LD = 1L << 21;  // 256 rows are within a buffer descriptor's 31-bit offsets
// A result that the products store themselves: 128 of its rows are within 32-bit offsets.
void check_result(const void* p, long ld, long rows, long width, const char* what) {
  check_matrix(p, ld, rows, width, what);
  require(rows <= 1 || ld < 1L << 24, what);
}

// ---- layer norm ----
void check_norm(const LayerNormArgs* a) {
  require(a, "no arguments");
  check_type(a->type);
  check_type(a->paramType);
  // the kernels read and write parameters as one of these two: another type has elements of another size
  require(a->paramType == a->type || a->paramType == DT_F32, "LayerNorm: paramType is neither type nor float32");
  require(a->rows >= 0 && a->rows < INT_MAX, "LayerNorm: bad number of rows");
  // (a long row's indices are ints that a workgroup's stride is added to)
  require(a->width >= 1 && a->width <= INT_MAX - 1024, "LayerNorm: bad width");
}
NormArgs norm_args(const LayerNormArgs* a) {
  NormArgs n{};
  n.x = a->x; n.ldx = a->ldx;
  n.weight = a->weight; n.bias = a->bias;
  n.mean = a->mean; n.rstd = a->rstd;
  n.rows = a->rows; n.width = a->width;
  n.dtype = a->type; n.param_dtype = a->paramType;
  n.eps = a->eps;
  return n;
}

// ---- gated block ----
void check_mlp(const GatedMLPArgs* a) {
  require(a, "no arguments");
  check_type(a->type);
  require(a->rows >= 0 && a->rows < MAX_ROWS, "GatedMLP: bad number of rows");
  require(a->width >= 1 && a->hidden >= 1 && a->width < MAX_LD && a->hidden < MAX_LD, "GatedMLP: bad width");
  require(a->act >= ACT_SILU && a->act <= ACT_CUBIC, "GatedMLP: unknown activation");
}
void check_mlp_tensors(const GatedMLPArgs* a) {
  check_matrix(a->x, a->ldx, a->rows, a->width, "GatedMLP: x");
  check_matrix(a->gate, a->ldgate, a->hidden, a->width, "GatedMLP: gate");
  check_matrix(a->up, a->ldup, a->hidden, a->width, "GatedMLP: up");
  check_matrix(a->down, a->lddown, a->width, a->hidden, "GatedMLP: down");
}
void set_act(ProductArgs& p, const GatedMLPArgs* a) {
  p.act = a->act;
  for (int i = 0; i < 4; i++) p.coef[i] = a->coef[i];
}

// A matrix as the products take it: where it is, or a copy in the workspace.
struct Held {
  const uint16_t* p;
  long ld, part;             // part: elements from one part to the next
  int parts = 1;             // three of a float32 matrix, two of a 16-bit intermediate of few rows
  const uint16_t* at(int k) const { return p + k * part; }
};
long up8(long n) { return (n + 7) & ~7L; }
bool fits(const void* p, long ld, long rows, long width, int type) {
  return type != DT_F32 && (uintptr_t)p % 16 == 0 && width % 8 == 0 && (rows <= 1 || ld % 8 == 0) && ld < MAX_LD;
}
// An intermediate of the operator's own.
Held hold(Arena& m, long rows, long width, int type, bool exact = false) {
  const long ld = up8(width), part = rows * ld;
  const int parts = type == DT_F32 ? 3 : exact ? 2 : 1;
  return {m.take<uint16_t>((size_t)part * parts), ld, parts > 1 ? part : 0, parts};
}
// Where a 16-bit operator has so few rows, its intermediates are held in two
// parts.  Rounded to one, each result has two roundings, sqrt(2) times the
// error of its own; over many rows that is what it stays, in a sum over few of
// them one value's rounding may be all there is (up to 2.5 times, seen 1.6).
// The products are bound by the weights there, not by the matrix units, and up
// to 64 rows are one step of k in the weights' gradients: 64 x 1,024 x 4,096,
// forward and backward, 81 us with two parts and 73 with one; the loss of 64 x
// 1,024 against 65,536 172 and 162.  The parts are of the operator's type, with
// its range: float16 hidden values and their gradients are infinite beyond 65504
// and lose bits below 2^-14 (a loss in float16 is scaled; dl is by itself).
// A teacher's few largest probabilities are most of dl, one or two values a row,
// of any number of rows: its rounding to one part is a rounding of what a table's row
// gets.  Two parts are kept up to 256 rows, a bound of cost alone.  Backward pass in
// bfloat16, one part and two (dx and dtable off by 0.0023-0.0024 and 0.0017): 94 x 172
// against 43,339 81 and 92 us, 256 x 1,024 against 65,536 197 and 275; 1,024 rows
// 469 and 723, 4,096 1,560 and 2,510.  A caller who needs the exact one has float32.
constexpr long FEW = 64, FEW_TAUGHT = 256;
bool few_rows(long rows, int type, long most = FEW) { return type != DT_F32 && rows <= most; }
// Matrices that are copied first, all in one launch: where alignment, an odd
// width or float32 does not let the tiles be loaded from a matrix itself.  A
// pass over it; a product of more than a few rows reads it many times.
struct Copies {
  LayOut j[8];
  int n = 0;
  const Held& add(const Held& h, const void* p, long ld, long rows, long width, const int* at = nullptr, const int* count = nullptr) {
    j[n++] = {p, ld, (void*)h.p, h.ld, h.part, at, count, rows, (int)width};
    return h;
  }
  Held held(Arena& m, const void* p, long ld, long rows, long width, int type, bool same_ld = true) {
    if (fits(p, ld, rows, width, type) && same_ld) return {(const uint16_t*)p, rows > 1 ? ld : width, 0, 1};
    return add(hold(m, rows, width, type), p, ld, rows, width);
  }
};
// The pairs of parts whose products make one product, smallest first: of three
// parts of 8 bits each those above 2^-24, of two parts of one factor both.  All
// but the last, the first parts', are corrections, and come before the last
// pairs of other products of the same sum.
int add_pairs(ProductArgs& p, const Held& a, const Held& b, const Held* b2 = nullptr) {
  static const int part_a[6] = {0, 1, 2, 0, 1, 0}, part_b[6] = {2, 1, 0, 1, 0, 0};
  const bool f32 = p.dtype == DT_F32;
  const int n = f32 ? 6 : std::max(a.parts, b.parts);
  for (int k = 0; k < n; k++) {
    const int ia = f32 ? part_a[k] : std::min(n - 1 - k, a.parts - 1), ib = f32 ? part_b[k] : std::min(n - 1 - k, b.parts - 1);
    const int at = k < n - 1 ? p.corrections++ : p.pairs;
    for (int i = p.pairs; i > at; i--) { p.a[i] = p.a[i - 1]; p.b[i] = p.b[i - 1]; }
    p.a[at] = a.at(ia);
    p.b[at] = b.at(ib);
    if (b2) p.b2[at] = b2->at(ib);   // (one product: none is moved)
    p.pairs++;
  }
  p.lda = a.ld; p.ldb = b.ld;
  return p.pairs;
}

// The scratch of the largest of an operator's products, which use it in turn.
float* scratch(Arena& m, std::initializer_list<size_t> sizes) { return (float*)m.bytes(std::max(sizes)); }

// Single vectors: two kernels that read the weights once.
size_t mlp_skinny(const GatedMLPArgs* a, bool count, hipStream_t st) {
  Arena m{count ? nullptr : (char*)a->workspace};
  const long ldh = up8(a->hidden);
  float* h = m.take<float>((size_t)a->rows * ldh);
  if (count) return m.used;
  SkinnyArgs p{};
  p.dtype = a->type;
  p.T = (int)a->rows; p.N = a->hidden; p.K = a->width;
  p.x = a->x; p.ldx = a->ldx;
  p.w = a->gate; p.ldw = a->ldgate;
  p.w2 = a->up; p.ldw2 = a->ldup;
  p.out = h; p.ldout = ldh;
  p.g = a->g; p.u = a->u; p.ldg = ldh;
  p.act = a->act;
  for (int i = 0; i < 4; i++) p.coef[i] = a->coef[i];
  skinny_gate(p, st);
  p.N = a->width; p.K = a->hidden;
  p.x = h; p.ldx = ldh;
  p.w = a->down; p.ldw = a->lddown;
  p.out = a->y; p.ldout = a->ldy;
  skinny_store(p, st);
  return m.used;
}

size_t mlp_forward(const GatedMLPArgs* a, bool count, hipStream_t st) {
  if (a->rows <= skinny_rows(a->type)) return mlp_skinny(a, count, st);
  Arena m{count ? nullptr : (char*)a->workspace};
  const int type = a->type;
  const bool same = a->ldgate == a->ldup;
  const bool few = few_rows(a->rows, type);
  const Held h = hold(m, a->rows, a->hidden, type, few);
  Copies copy;
  const Held x = copy.held(m, a->x, a->ldx, a->rows, a->width, type);
  const Held gate = copy.held(m, a->gate, a->ldgate, a->hidden, a->width, type, same && fits(a->up, a->ldup, a->hidden, a->width, type));
  const Held up = copy.held(m, a->up, a->ldup, a->hidden, a->width, type, same && fits(a->gate, a->ldgate, a->hidden, a->width, type));
  const Held down = copy.held(m, a->down, a->lddown, a->width, a->hidden, type);
  const int parts = type == DT_F32 ? 6 : 1;
  float* partial = scratch(m, {product_scratch({{a->rows, a->hidden}}, a->width, parts, true),
                               product_scratch({{a->rows, a->width}}, a->hidden, parts * (few ? 2 : 1))});
  if (count) return m.used;
  lay_out(copy.j, copy.n, type, st);
  ProductArgs p{};
  p.dtype = type;
  p.M = (int)a->rows; p.N = a->hidden; p.K = a->width;
  add_pairs(p, x, gate, &up);
  p.g = a->g; p.u = a->u; p.h = (void*)h.p; p.ldh = h.ld; p.hpart = h.part;
  p.partial = partial;
  set_act(p, a);
  product_gate(p, st);
  ProductArgs q{};
  q.dtype = q.ctype = type;
  q.M = (int)a->rows; q.N = a->width; q.K = a->hidden;
  add_pairs(q, h, down);
  q.partial = partial;
  q.c = a->y; q.ldc = a->ldy;
  product_nt(q, st);
  return m.used;
}

size_t mlp_backward(const GatedMLPArgs* a, bool count, hipStream_t st) {
  Arena m{count ? nullptr : (char*)a->workspace};
  const int type = a->type;
  const bool same = a->ldgate == a->ldup;
  const bool few = few_rows(a->rows, type);
  const Held dg = hold(m, a->rows, a->hidden, type, few), du = hold(m, a->rows, a->hidden, type, few), h = hold(m, a->rows, a->hidden, type, few);
  Copies copy;
  const Held x = copy.held(m, a->x, a->ldx, a->rows, a->width, type), dy = copy.held(m, a->dy, a->lddy, a->rows, a->width, type);
  const Held gate = copy.held(m, a->gate, a->ldgate, a->hidden, a->width, type, same && fits(a->up, a->ldup, a->hidden, a->width, type));
  const Held up = copy.held(m, a->up, a->ldup, a->hidden, a->width, type, same && fits(a->gate, a->ldgate, a->hidden, a->width, type));
  const Held down = copy.held(m, a->down, a->lddown, a->width, a->hidden, type);
  const int parts = type == DT_F32 ? 6 : 1;
  const Shape in{a->hidden, a->width}, out{a->width, a->hidden};
  const int held = parts * (few ? 2 : 1);   // pairs of a product with an intermediate
  float* partial = scratch(m, {product_scratch({{a->rows, a->hidden}}, a->width, parts), product_scratch({{a->rows, a->width}}, a->hidden, 2 * held),
                               product_scratch({in, in, out}, a->rows, held)});
  if (count) return m.used;
  lay_out(copy.j, copy.n, type, st);
  // dh = dy down, and through the product and the activation
  ProductArgs p{};
  p.dtype = type;
  p.M = (int)a->rows; p.N = a->hidden; p.K = a->width;
  add_pairs(p, dy, down);
  p.g = a->g; p.u = a->u; p.h = (void*)h.p; p.dg = (void*)dg.p; p.du = (void*)du.p; p.ldh = h.ld; p.hpart = h.part;
  p.partial = partial;
  set_act(p, a);
  product_gate_grad(p, st);
  // dx = dg gate + du up
  ProductArgs q{};
  q.dtype = q.ctype = type;
  q.M = (int)a->rows; q.N = a->width; q.K = a->hidden;
  add_pairs(q, dg, gate);
  add_pairs(q, du, up);
  q.partial = partial;
  q.c = a->dx; q.ldc = a->lddx;
  product_nn(q, st);
  // the weights' gradients: sums over the rows
  auto weight = [&](const Held& l, const Held& r, const Shape& s, void* to) {
    ProductArgs w{};
    w.dtype = w.ctype = type;
    w.M = (int)s.M; w.N = (int)s.N; w.K = (int)a->rows;
    add_pairs(w, l, r);
    w.partial = partial;
    w.c = to; w.ldc = s.N;
    return w;
  };
  product_tn(weight(dg, x, in, a->dgate), weight(du, x, in, a->dup), weight(dy, h, out, a->ddown), st);
  return m.used;
}

// ---- cross entropy ----
void check_ce(const CrossEntropyArgs* a) {
  require(a, "no arguments");
  check_type(a->type);
  require(a->rows >= 0 && a->rows < MAX_ROWS, "CrossEntropy: bad number of rows");
  require(a->width >= 1 && a->width < MAX_LD, "CrossEntropy: bad width");
  require(a->vocab >= 1, "CrossEntropy: bad number of table rows");
}
void check_ce_tensors(const CrossEntropyArgs* a) {
  check_matrix(a->x, a->ldx, a->rows, a->width, "CrossEntropy: x");
  check_matrix(a->table, a->ldtable, a->vocab, a->width, "CrossEntropy: table");
  require(a->target || !a->rows, "CrossEntropy: target");
  require(a->lse || !a->rows, "CrossEntropy: lse");
}

size_t ce_skinny(const CrossEntropyArgs* a, bool count, hipStream_t st) {
  Arena m{count ? nullptr : (char*)a->workspace};
  SkinnyArgs p{};
  p.dtype = a->type;
  p.T = (int)a->rows; p.N = a->vocab; p.K = a->width;
  p.x = a->x; p.ldx = a->ldx;
  p.w = a->table; p.ldw = a->ldtable;
  p.target = a->target;
  p.picked = m.take<float>(a->rows);
  p.part = m.take<float2>((size_t)a->rows * skinny_softmax_parts(a->vocab));
  if (count) return m.used;
  skinny_softmax(p, a->ignore, a->loss, a->lse, st);
  return m.used;
}

size_t ce_forward(const CrossEntropyArgs* a, bool count, hipStream_t st) {
  if (a->rows <= skinny_rows(a->type)) return ce_skinny(a, count, st);
  Arena m{count ? nullptr : (char*)a->workspace};
  const long n = a->rows;
  const clr::SoftmaxPlan plan = clr::softmax_plan(n, a->vocab, a->width, a->type == DT_F32 ? 6 : 1);
  RowsArgs r{a->target, nullptr, n, a->ignore, a->vocab};
  r.rows = m.take<int>(n); r.tgt = m.take<int>(n); r.count = m.take<int>(1);
  r.picked = m.take<float>(n); r.loss = a->loss; r.lse = a->lse;
  const Held x = hold(m, n, a->width, a->type);
  float2* part = m.take<float2>((size_t)n * plan.parts);
  Copies copy;
  copy.add(x, a->x, a->ldx, n, a->width, r.rows, r.count);
  const Held table = copy.held(m, a->table, a->ldtable, a->vocab, a->width, a->type);
  if (count) return m.used;
  kept_rows(r, st);
  lay_out(copy.j, copy.n, a->type, st);
  ProductArgs p{};
  p.dtype = a->type;
  p.M = (int)n; p.N = a->vocab; p.K = a->width;
  add_pairs(p, x, table);
  p.count = r.count; p.target = r.tgt; p.picked = r.picked; p.part = part;
  product_softmax(p, plan, st);
  softmax_finish(part, plan.parts, r.picked, r.rows, r.count, n, a->loss, a->lse, st);
  return m.used;
}

// Rows of the table whose gradients of the logits are held at a time: those
// of all rows of x take at most 256 MiB, what the last-level cache holds, or
// there are 1,024 of them.
constexpr long PIECE_BYTES = 256L << 20;
static_assert(PIECE_BYTES < 1L << 31 && 256 * 1024 * 2 < 1L << 31, "the rows of a tile of dl are within 31-bit offsets, whatever their number and width");
int piece_rows(long rows, int vocab, int type, bool few) {
  const long most = PIECE_BYTES / (std::max<long>(rows, 1) * (type == DT_F32 ? 6 : few ? 4 : 2));
  return (int)std::min<long>(up8(vocab), std::max<long>(1024, most / 1024 * 1024));
}

// The gradients of a loss against a table, dx = dl table and dtable = dl^T x, from `logits_grad`, which leaves dl for
// some of the table's rows.  The arguments' targets and gradients, of which `r` says which.
template <class Args, class F> size_t table_backward(const Args* a, RowsArgs r, bool few, int most, bool count, hipStream_t st, F&& logits_grad) {
  Arena m{count ? nullptr : (char*)a->workspace};
  const long n = a->rows, D = a->width;
  const int piece = piece_rows(a->rows, a->vocab, a->type, few);
  r.rows = m.take<int>(n); r.tgt = m.take<int>(n); r.place = m.take<int>(n); r.count = m.take<int>(1);
  float* scale = m.take<float>(1);
  if (a->type == DT_F16) r.scale = scale;
  r.lse = a->lse; r.lse_kept = m.take<float>(n); r.grad_kept = m.take<float>(n);
  const Held x = hold(m, n, a->width, a->type), dl = hold(m, n, piece, a->type, few);
  // two parts are twice as many rows for dx, in a tile that has room for them (the table is read once); scatter_rows adds them
  const long stacked = few ? 2 * n : n;
  float* acc = m.take<float>((size_t)stacked * D);
  const int parts = a->type == DT_F32 ? 6 : 1, sums = parts * (few ? 2 : 1), last = a->vocab % piece ? a->vocab % piece : piece;
  float* partial = scratch(m, {product_scratch({{stacked, D}}, piece, parts, false, most), product_scratch({{stacked, D}}, last, parts, false, most),
                               product_scratch({{piece, D}}, n, sums), product_scratch({{last, D}}, n, sums)});
  Copies copy;
  copy.add(x, a->x, a->ldx, n, a->width, r.rows, r.count);
  const Held table = copy.held(m, a->table, a->ldtable, a->vocab, a->width, a->type);
  if (count) return m.used;
  kept_rows(r, st);
  lay_out(copy.j, copy.n, a->type, st);
  for (long v0 = 0; v0 < a->vocab; v0 += piece) {
    const int len = (int)std::min<long>(piece, a->vocab - v0);
    const Held rows{table.p + v0 * table.ld, table.ld, table.part, table.parts};
    ProductArgs p{};
    p.dtype = a->type; p.count = r.count;
    p.M = (int)n; p.N = len; p.K = a->width;
    add_pairs(p, x, rows);
    p.c = (void*)dl.p; p.ldc = dl.ld; p.hpart = dl.part;
    p.n0 = (int)v0; p.target = r.tgt; p.lse = r.lse_kept; p.grad = r.grad_kept; p.scale = r.scale;
    logits_grad(p, r, dl);
    ProductArgs q{};
    q.dtype = a->type; q.ctype = DT_F32; q.count = few ? nullptr : r.count;   // (few: rows past the count are anything, and are not looked at)
    q.M = (int)stacked; q.N = a->width; q.K = len;
    add_pairs(q, {dl.p, dl.ld, dl.part, few ? 1 : dl.parts}, rows);
    q.partial = partial;
    q.most = most;
    q.c = acc; q.ldc = D; q.add = v0 > 0;
    product_nn(q, st);
    ProductArgs w{};
    w.dtype = w.ctype = a->type; w.count = r.count; w.count_k = true;
    w.M = len; w.N = a->width; w.K = (int)n;
    add_pairs(w, dl, x);
    w.partial = partial;
    w.c = (char*)a->dtable + v0 * D * dtype_size(a->type); w.ldc = D;
    w.unscale = r.scale;
    product_tn(w, st);
  }
  scatter_rows(acc, D, few ? n * D : 0, r.place, r.scale, a->dx, a->lddx, n, a->width, a->type, st);
  return m.used;
}

size_t ce_backward(const CrossEntropyArgs* a, bool count, hipStream_t st) {
  return table_backward(a, RowsArgs{a->target, a->dloss, a->rows, a->ignore, a->vocab}, few_rows(a->rows, a->type), clr::SPLITS, count, st,
                        [&](const ProductArgs& p, const RowsArgs&, const Held&) { product_softmax_grad(p, st); });
}

// ---- distillation ----
void check_teach(const DistillationArgs* a) {
  require(a, "no arguments");
  check_type(a->type);
  check_type(a->teacherType);
  require(a->teacherType == a->type || a->teacherType == DT_F32, "Distillation: teacherType is neither type nor float32");
  require(a->rows >= 0 && a->rows < MAX_ROWS, "Distillation: bad number of rows");
  require(a->width >= 1 && a->width < MAX_LD, "Distillation: bad width");
  require(a->vocab >= 1, "Distillation: bad number of table rows");
  require(a->top >= 1 && a->top <= MOST_TOP, "Distillation: bad number of a teacher's logits");
  // (its square is a factor of the loss, its reciprocal of the logits)
  require(a->temperature >= 0x1p-60f && a->temperature <= 0x1p60f, "Distillation: bad temperature");
}
void check_teach_tensors(const DistillationArgs* a) {
  check_matrix(a->x, a->ldx, a->rows, a->width, "Distillation: x");
  check_matrix(a->table, a->ldtable, a->vocab, a->width, "Distillation: table");
  require(a->lse || !a->rows, "Distillation: lse");
  require((a->kept && a->scores && a->probs && a->cols) || !a->rows, "Distillation: kept, scores, probs and cols");
}

// Whether the entries' scores are picked out of the product's tiles, or
// computed from the table's rows.  Microseconds, measured: the rows at 3.4 TB/s
// (a common one comes from the caches); two launches more and the order of the
// entries, each compared with each, the end of a tile 1.6, a row's entries of a
// tile one after another 0.4.  8,192 x 2,048 against 131,072 rows, 64 entries,
// bfloat16, both directions: 14,290 picked, 14,885 computed; 192 x 560 against
// 448, 104 entries, the forward kernels: 74 and 38.
bool teach_picks(const DistillationArgs* a) {
  const double rows = (double)a->rows, top = a->top, across = (double)clr::ceil_div(a->vocab, 256);
  const double computed = rows * top * a->width * dtype_size(a->type) / 3.4e6 + 5e-7 * rows * top * top;
  const double picked = 12 + (3.4e-4 + 1e-6 * rows) * top * top + 1.6 * (double)clr::ceil_div(a->rows, 256) * across / 256 + 0.4 * top / across;
  return computed > picked;
}

size_t teach_forward(const DistillationArgs* a, bool count, hipStream_t st) {
  Arena m{count ? nullptr : (char*)a->workspace};
  const long n = a->rows;
  const float rate = 1.0f / a->temperature;
  TeachArgs e{};
  e.x = a->x; e.ldx = a->ldx;
  e.table = a->table; e.ldtable = a->ldtable;
  e.ids = a->ids; e.logits = a->logits;
  e.scores = a->scores; e.probs = a->probs; e.cols = a->cols;
  e.kept = a->kept;
  e.rows = n; e.width = a->width; e.vocab = a->vocab; e.top = a->top;
  e.dtype = a->type; e.teacher_type = a->teacherType;
  e.ignore = a->ignore;
  e.temperature = a->temperature;
  e.parts = n ? entry_parts(n, a->top) : 1;
  TeachFinish f{};
  f.scores = a->scores; f.probs = a->probs; f.kept = a->kept;
  f.loss = a->loss; f.lse = a->lse;
  f.n = n; f.top = a->top;
  f.temperature = a->temperature;
  if (n <= skinny_rows(a->type)) {
    SkinnyArgs p{};
    p.dtype = a->type;
    p.T = (int)n; p.N = a->vocab; p.K = a->width;
    p.x = a->x; p.ldx = a->ldx;
    p.w = a->table; p.ldw = a->ldtable;
    p.rate = rate;
    f.parts = skinny_softmax_parts(a->vocab);
    f.part = p.part = m.take<float2>((size_t)n * f.parts);
    if (count) return m.used;
    skinny_teach(p, e, st);
    teach_finish(f, st);
    return m.used;
  }
  const clr::SoftmaxPlan plan = clr::softmax_plan(n, a->vocab, a->width, a->type == DT_F32 ? 6 : 1);
  RowsArgs r{a->kept, nullptr, n, TEACH_NONE, TEACH_OUTSIDE};
  r.rows = m.take<int>(n); r.tgt = m.take<int>(n); r.count = m.take<int>(1);
  r.loss = a->loss; r.lse = a->lse;
  const Held x = hold(m, n, a->width, a->type);
  float2* part = m.take<float2>((size_t)n * plan.parts);
  const bool picks = teach_picks(a);
  if (picks) {
    e.starts = m.take<uint16_t>((size_t)n * (plan.parts + 1));
    e.tiles = plan.parts;
    e.shift = plan.plan.big ? 8 : 7;
    e.which = r.rows; e.count = r.count;
  }
  Copies copy;
  copy.add(x, a->x, a->ldx, n, a->width, r.rows, r.count);
  const Held table = copy.held(m, a->table, a->ldtable, a->vocab, a->width, a->type);
  if (count) return m.used;
  if (picks) teach_kept(e, st);
  else teach_entries(e, st);
  kept_rows(r, st);
  if (picks) teach_order(e, st);
  lay_out(copy.j, copy.n, a->type, st);
  ProductArgs p{};
  p.dtype = a->type;
  p.M = (int)n; p.N = a->vocab; p.K = a->width;
  add_pairs(p, x, table);
  p.count = r.count; p.part = part;
  p.rate = rate;
  p.starts = e.starts; p.ldstarts = plan.parts + 1;
  p.rows = r.rows; p.cols = a->cols; p.scores = a->scores; p.top = a->top;
  product_teach(p, plan, st);
  f.part = part; f.parts = plan.parts;
  f.rows = r.rows; f.count = r.count;
  teach_finish(f, st);
  return m.used;
}

size_t teach_backward(const DistillationArgs* a, bool count, hipStream_t st) {
  RowsArgs r{a->kept, a->dloss, a->rows, TEACH_NONE, TEACH_OUTSIDE};
  r.factor = a->temperature;
  return table_backward(a, r, few_rows(a->rows, a->type, FEW_TAUGHT), clr::MANY_SPLITS, count, st, [&](ProductArgs p, const RowsArgs& r, const Held& dl) {
    p.rate = 1.0f / a->temperature;
    product_teach_grad(p, st);
    TeachPatch t{};
    t.dl = (uint16_t*)dl.p; t.ld = dl.ld; t.part = dl.part;
    t.rows = r.rows; t.tgt = r.tgt; t.count = r.count;
    t.lse = r.lse_kept; t.grad = r.grad_kept; t.scale = r.scale;
    t.cols = a->cols; t.scores = a->scores; t.probs = a->probs;
    t.n = a->rows; t.top = a->top; t.dtype = a->type;
    t.v0 = p.n0; t.len = p.N;
    teach_patch(t, st);
  });
}

void check_total(const LossTotalArgs* a) {
  require(a, "no arguments");
  require(a->rows >= 0 && a->rows < MAX_ROWS, "LossTotal: bad number of rows");
}

// ---- embedding ----
void check_embedding(const EmbeddingArgs* a) {
  require(a, "no arguments");
  check_type(a->type);
  require(a->tokens >= 0 && a->tokens < MAX_ROWS, "Embedding: bad number of tokens");
  // (indices of a row's elements are ints)
  require(a->width >= 1 && a->width <= INT_MAX - 1024, "Embedding: bad width");
  require(a->vocab >= 1, "Embedding: bad number of table rows");
}
EmbedArgs embed_args(const EmbeddingArgs* a) {
  EmbedArgs e{};
  e.ids = a->ids;
  e.tokens = a->tokens; e.width = a->width; e.vocab = a->vocab;
  e.ignore = a->ignore;
  e.dtype = a->type;
  e.scale = a->scale;
  return e;
}
size_t embedding_space(const EmbeddingArgs* a) { return embedding_grad_workspace(a->tokens, a->width, a->vocab, a->type); }

// ---- preference ----
constexpr long MAX_LINE = 1L << 40;
void check_pairs(const PreferenceArgs* a) {
  require(a, "no arguments");
  require(a->pairs >= 0 && a->pairs < MAX_ROWS, "Preference: bad number of pairs");
  require(a->length >= 0 && a->length <= MAX_LINE, "Preference: bad length");
  require(a->kind == PAIR_LOGISTIC || a->kind == PAIR_HINGE, "Preference: unknown kind");
  require(a->beta - a->beta == 0.0f && a->margin - a->margin == 0.0f, "Preference: beta and margin are not finite");
  require(a->smoothing >= 0.0f && a->smoothing <= (a->kind == PAIR_LOGISTIC ? 1.0f : 0.0f), "Preference: bad smoothing");
}
// A line of tokens, or a matrix of them.
void check_tokens(const PreferenceArgs* a, const void* p, long ld, const char* what) {
  const bool any = a->length && (a->offsets || a->pairs);
  require(p || !any, what);
  require(a->offsets || a->pairs == 0 || ld >= a->length, what);
}
PairArgs pair_args(const PreferenceArgs* a) {
  PairArgs p{};
  p.target = a->target; p.ldtarget = a->ldtarget;
  p.offsets = a->offsets;
  p.slope = a->slope;
  p.pairs = a->pairs; p.length = a->length;
  p.ignore = a->ignore;
  return p;
}

template <class F> long sized(F&& f) {
  try { return (long)f(); } catch (const std::exception& e) { return report_error(e.what()); }
}

}  // namespace

extern "C" {

int LayerNorm(const LayerNormArgs* a, void* stream) {
  return clr::guarded([&] {
    check_norm(a);
    check_matrix(a->x, a->ldx, a->rows, a->width, "LayerNorm: x");
    check_matrix(a->y, a->ldy, a->rows, a->width, "LayerNorm: y");
    require(a->weight, "LayerNorm: weight");
    NormArgs n = norm_args(a);
    n.y = a->y; n.ldy = a->ldy;
    norm_forward_launch(n, (hipStream_t)stream);
  });
}
long LayerNormGradWorkspace(const LayerNormArgs* a) {
  return sized([&] { check_norm(a); return norm_backward_workspace(a->rows, a->width); });
}
int LayerNormGrad(const LayerNormArgs* a, void* stream) {
  return clr::guarded([&] {
    check_norm(a);
    check_matrix(a->x, a->ldx, a->rows, a->width, "LayerNormGrad: x");
    check_matrix(a->dy, a->lddy, a->rows, a->width, "LayerNormGrad: dy");
    check_matrix(a->dx, a->lddx, a->rows, a->width, "LayerNormGrad: dx");
    require(a->weight && a->dweight, "LayerNormGrad: weight");
    require((a->mean && a->rstd) || !a->rows, "LayerNormGrad: mean and rstd");
    check_space(a->workspace, a->workspaceBytes, norm_backward_workspace(a->rows, a->width));
    NormArgs n = norm_args(a);
    n.y = const_cast<void*>(a->dy); n.ldy = a->lddy;
    n.dx = a->dx; n.lddx = a->lddx;
    n.dweight = a->dweight; n.dbias = a->dbias;
    n.workspace = a->workspace;
    norm_backward_launch(n, (hipStream_t)stream);
  });
}

long GatedMLPWorkspace(const GatedMLPArgs* a) {
  return sized([&] { check_mlp(a); return mlp_forward(a, true, nullptr); });
}
int GatedMLP(const GatedMLPArgs* a, void* stream) {
  return clr::guarded([&] {
    check_mlp(a);
    check_mlp_tensors(a);
    check_result(a->y, a->ldy, a->rows, a->width, "GatedMLP: y");
    require(!a->g == !a->u, "GatedMLP: g and u are kept together");
    require(((uintptr_t)a->g | (uintptr_t)a->u) % 16 == 0, "GatedMLP: g and u are not aligned to 16 bytes");
    if (!a->rows) return;
    check_space(a->workspace, a->workspaceBytes, mlp_forward(a, true, nullptr));
    mlp_forward(a, false, (hipStream_t)stream);
  });
}
long GatedMLPGradWorkspace(const GatedMLPArgs* a) {
  return sized([&] { check_mlp(a); return mlp_backward(a, true, nullptr); });
}
int GatedMLPGrad(const GatedMLPArgs* a, void* stream) {
  return clr::guarded([&] {
    check_mlp(a);
    check_mlp_tensors(a);
    check_matrix(a->dy, a->lddy, a->rows, a->width, "GatedMLPGrad: dy");
    check_result(a->dx, a->lddx, a->rows, a->width, "GatedMLPGrad: dx");
    require((a->g && a->u) || !a->rows, "GatedMLPGrad: g and u");
    require(((uintptr_t)a->g | (uintptr_t)a->u) % 16 == 0, "GatedMLPGrad: g and u are not aligned to 16 bytes");
    require(a->dgate && a->dup && a->ddown, "GatedMLPGrad: the weights' gradients");
    const size_t n = (size_t)a->width * a->hidden * dtype_size(a->type);
    if (!a->rows) {
      for (void* p : {a->dgate, a->dup, a->ddown}) fill_zero(p, n, (hipStream_t)stream);
      return;
    }
    check_space(a->workspace, a->workspaceBytes, mlp_backward(a, true, nullptr));
    mlp_backward(a, false, (hipStream_t)stream);
  });
}

long CrossEntropyWorkspace(const CrossEntropyArgs* a) {
  return sized([&] { check_ce(a); return ce_forward(a, true, nullptr); });
}
int CrossEntropy(const CrossEntropyArgs* a, void* stream) {
  return clr::guarded([&] {
    check_ce(a);
    check_ce_tensors(a);
    require(a->loss || !a->rows, "CrossEntropy: loss");
    if (!a->rows) return;
    check_space(a->workspace, a->workspaceBytes, ce_forward(a, true, nullptr));
    ce_forward(a, false, (hipStream_t)stream);
  });
}
long CrossEntropyGradWorkspace(const CrossEntropyArgs* a) {
  return sized([&] { check_ce(a); return ce_backward(a, true, nullptr); });
}
int CrossEntropyGrad(const CrossEntropyArgs* a, void* stream) {
  return clr::guarded([&] {
    check_ce(a);
    check_ce_tensors(a);
    check_matrix(a->dx, a->lddx, a->rows, a->width, "CrossEntropyGrad: dx");
    require(a->dtable, "CrossEntropyGrad: dtable");
    require(a->dloss || !a->rows, "CrossEntropyGrad: dloss");
    if (!a->rows) {
      fill_zero(a->dtable, (size_t)a->vocab * a->width * dtype_size(a->type), (hipStream_t)stream);
      return;
    }
    check_space(a->workspace, a->workspaceBytes, ce_backward(a, true, nullptr));
    ce_backward(a, false, (hipStream_t)stream);
  });
}

long DistillationWorkspace(const DistillationArgs* a) {
  return sized([&] { check_teach(a); return teach_forward(a, true, nullptr); });
}
int Distillation(const DistillationArgs* a, void* stream) {
  return clr::guarded([&] {
    check_teach(a);
    check_teach_tensors(a);
    require(a->ids || !a->rows, "Distillation: ids");
    require(a->logits || !a->rows, "Distillation: logits");
    require(a->loss || !a->rows, "Distillation: loss");
    if (!a->rows) return;
    check_space(a->workspace, a->workspaceBytes, teach_forward(a, true, nullptr));
    teach_forward(a, false, (hipStream_t)stream);
  });
}
long DistillationGradWorkspace(const DistillationArgs* a) {
  return sized([&] { check_teach(a); return teach_backward(a, true, nullptr); });
}
int DistillationGrad(const DistillationArgs* a, void* stream) {
  return clr::guarded([&] {
    check_teach(a);
    check_teach_tensors(a);
    check_matrix(a->dx, a->lddx, a->rows, a->width, "DistillationGrad: dx");
    require(a->dtable, "DistillationGrad: dtable");
    require(a->dloss || !a->rows, "DistillationGrad: dloss");
    if (!a->rows) {
      fill_zero(a->dtable, (size_t)a->vocab * a->width * dtype_size(a->type), (hipStream_t)stream);
      return;
    }
    check_space(a->workspace, a->workspaceBytes, teach_backward(a, true, nullptr));
    teach_backward(a, false, (hipStream_t)stream);
  });
}

long LossTotalWorkspace(const LossTotalArgs* a) {
  return sized([&] { check_total(a); return loss_total_bytes(a->rows); });
}
int LossTotal(const LossTotalArgs* a, void* stream) {
  return clr::guarded([&] {
    check_total(a);
    require(a->loss || !a->rows, "LossTotal: loss");
    require(a->total && a->factor, "LossTotal: total and factor");
    check_space(a->workspace, a->workspaceBytes, loss_total_bytes(a->rows));
    loss_total(a->loss, a->target, a->ignore, a->rows, a->workspace, a->total, a->factor, (hipStream_t)stream);
  });
}

long PreferenceWorkspace(const PreferenceArgs* a) {
  return sized([&] { check_pairs(a); return preference_workspace(a->pairs, a->length, a->offsets); });
}
int Preference(const PreferenceArgs* a, void* stream) {
  return clr::guarded([&] {
    check_pairs(a);
    check_tokens(a, a->loss, a->ldloss, "Preference: loss");
    if (a->reference) check_tokens(a, a->reference, a->ldreference, "Preference: reference");
    if (a->target) check_tokens(a, a->target, a->ldtarget, "Preference: target");
    require((a->value && a->ratio && a->slope) || !a->pairs, "Preference: value, ratio and slope");
    check_space(a->workspace, a->workspaceBytes, preference_workspace(a->pairs, a->length, a->offsets));
    if (!a->pairs) return;
    PairArgs p = pair_args(a);
    p.loss = a->loss; p.ldloss = a->ldloss;
    p.reference = a->reference; p.ldreference = a->ldreference;
    p.value = a->value; p.ratio = a->ratio; p.kept = a->kept;
    p.workspace = a->workspace;
    p.kind = a->kind; p.average = a->average;
    p.beta = a->beta; p.margin = a->margin; p.smoothing = a->smoothing;
    preference_launch(p, (hipStream_t)stream);
  });
}
int PreferenceGrad(const PreferenceArgs* a, void* stream) {
  return clr::guarded([&] {
    check_pairs(a);
    check_tokens(a, a->dloss, a->lddloss, "PreferenceGrad: dloss");
    if (a->target) check_tokens(a, a->target, a->ldtarget, "PreferenceGrad: target");
    require((a->slope && a->dvalue) || !a->pairs, "PreferenceGrad: slope and dvalue");
    if (!a->length || (!a->pairs && !a->offsets)) return;
    PairArgs p = pair_args(a);
    p.dvalue = a->dvalue;
    p.dloss = a->dloss; p.lddloss = a->lddloss;
    preference_grad_launch(p, (hipStream_t)stream);
  });
}

int Embedding(const EmbeddingArgs* a, void* stream) {
  return clr::guarded([&] {
    check_embedding(a);
    require(a->ids || !a->tokens, "Embedding: ids");
    check_matrix(a->table, a->ldtable, a->vocab, a->width, "Embedding: table");
    check_matrix(a->y, a->ldy, a->tokens, a->width, "Embedding: y");
    EmbedArgs e = embed_args(a);
    e.table = a->table; e.ldtable = a->ldtable;
    e.y = a->y; e.ldy = a->ldy;
    embedding_launch(e, (hipStream_t)stream);
  });
}
long EmbeddingGradWorkspace(const EmbeddingArgs* a) {
  return sized([&] { check_embedding(a); return embedding_space(a); });
}
int EmbeddingGrad(const EmbeddingArgs* a, void* stream) {
  return clr::guarded([&] {
    check_embedding(a);
    require(a->ids || !a->tokens, "EmbeddingGrad: ids");
    check_matrix(a->dy, a->lddy, a->tokens, a->width, "EmbeddingGrad: dy");
    require(a->dtable, "EmbeddingGrad: dtable");
    check_space(a->workspace, a->workspaceBytes, embedding_space(a));
    EmbedArgs e = embed_args(a);
    e.y = const_cast<void*>(a->dy); e.ldy = a->lddy;
    e.dtable = a->dtable;
    e.workspace = a->workspace;
    embedding_grad_launch(e, (hipStream_t)stream);
  });
}

}  // extern "C"
