// cleartext.hip -- C ABI of the operators that train and score in the clear:
// argument checks, the division of a workspace, and the order of the launches.
#include <algorithm>
#include <climits>
#include "cleartext.h"
#include "norm.h"
#include "products.h"
#include "skinny.h"
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
bool few_rows(long rows, int type) { return type != DT_F32 && rows <= 64; }
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
int piece_rows(const CrossEntropyArgs* a) {
  const long most = PIECE_BYTES / (std::max<long>(a->rows, 1) * (a->type == DT_F32 ? 6 : few_rows(a->rows, a->type) ? 4 : 2));
  return (int)std::min<long>(up8(a->vocab), std::max<long>(1024, most / 1024 * 1024));
}

size_t ce_backward(const CrossEntropyArgs* a, bool count, hipStream_t st) {
  Arena m{count ? nullptr : (char*)a->workspace};
  const long n = a->rows, D = a->width;
  const int piece = piece_rows(a);
  RowsArgs r{a->target, a->dloss, n, a->ignore, a->vocab};
  r.rows = m.take<int>(n); r.tgt = m.take<int>(n); r.place = m.take<int>(n); r.count = m.take<int>(1);
  float* scale = m.take<float>(1);
  if (a->type == DT_F16) r.scale = scale;
  r.lse = a->lse; r.lse_kept = m.take<float>(n); r.grad_kept = m.take<float>(n);
  const bool few = few_rows(n, a->type);
  const Held x = hold(m, n, a->width, a->type), dl = hold(m, n, piece, a->type, few);
  // two parts are twice as many rows for dx, in a tile that has room for them (the table is read once); scatter_rows adds them
  const long stacked = few ? 2 * n : n;
  float* acc = m.take<float>((size_t)stacked * D);
  const int parts = a->type == DT_F32 ? 6 : 1, sums = parts * (few ? 2 : 1), last = a->vocab % piece ? a->vocab % piece : piece;
  float* partial = scratch(m, {product_scratch({{stacked, D}}, piece, parts), product_scratch({{stacked, D}}, last, parts),
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
    product_softmax_grad(p, st);
    ProductArgs q{};
    q.dtype = a->type; q.ctype = DT_F32; q.count = few ? nullptr : r.count;   // (few: rows past the count are anything, and are not looked at)
    q.M = (int)stacked; q.N = a->width; q.K = len;
    add_pairs(q, {dl.p, dl.ld, dl.part, few ? 1 : dl.parts}, rows);
    q.partial = partial;
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

void check_total(const LossTotalArgs* a) {
  require(a, "no arguments");
  require(a->rows >= 0 && a->rows < MAX_ROWS, "LossTotal: bad number of rows");
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

}  // extern "C"
