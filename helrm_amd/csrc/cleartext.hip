// cleartext.hip -- C ABI of the operators that train and score in the clear:
// argument checks, the division of a workspace, and the order of the launches.
#include <algorithm>
#include <climits>
#include "cleartext.h"
#include "norm.h"
#include "products.h"
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
// Rows of a matrix: the tiles' row count fits a launch, and a row's stride covers it.
void check_matrix(const void* p, long ld, long rows, long width, const char* what) {
  require(p || !rows, what);
  require(rows <= 1 || ld >= width, what);
}
constexpr long MAX_ROWS = 4L << 20;  // 65,535 tiles of 64

// ---- layer norm ----
void check_norm(const LayerNormArgs* a) {
  require(a, "no arguments");
  check_type(a->type);
  check_type(a->paramType);
  require(a->rows >= 0 && a->rows < INT_MAX, "LayerNorm: bad number of rows");
  require(a->width >= 1, "LayerNorm: bad width");
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
  require(a->width >= 1 && a->hidden >= 1 && a->width < MAX_ROWS && a->hidden < MAX_ROWS, "GatedMLP: bad width");
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

size_t mlp_forward(const GatedMLPArgs* a, void* ws, hipStream_t st) {
  Arena m{(char*)ws};
  const long F = a->hidden;
  void* h = m.bytes((size_t)a->rows * F * dtype_size(a->type));
  if (!ws) return m.used;
  ProductArgs p{};
  p.dtype = a->type;
  p.M = (int)a->rows; p.N = a->hidden; p.K = a->width; p.pairs = 1;
  p.a[0] = {a->x, a->ldx, 1};
  p.b[0] = {a->gate, a->ldgate, 1};
  p.b[1] = {a->up, a->ldup, 1};
  p.g = a->g; p.u = a->u; p.h = h;
  set_act(p, a);
  product_gate(p, st);
  ProductArgs q{};
  q.dtype = q.ctype = a->type;
  q.M = (int)a->rows; q.N = a->width; q.K = a->hidden; q.pairs = 1;
  q.a[0] = {h, F, 1};
  q.b[0] = {a->down, a->lddown, 1};
  q.c = a->y; q.ldc = a->ldy;
  product_store(q, st);
  return m.used;
}

size_t mlp_backward(const GatedMLPArgs* a, void* ws, hipStream_t st) {
  Arena m{(char*)ws};
  const long F = a->hidden, D = a->width;
  const size_t n = (size_t)a->rows * F * dtype_size(a->type);
  void* dg = m.bytes(n); void* du = m.bytes(n); void* h = m.bytes(n);
  if (!ws) return m.used;
  ProductArgs p{};
  p.dtype = p.ctype = a->type;
  // dh = dy down, and through the product and the activation
  p.M = (int)a->rows; p.N = a->hidden; p.K = a->width; p.pairs = 1;
  p.a[0] = {a->dy, a->lddy, 1};
  p.b[0] = {a->down, 1, a->lddown};
  p.g = a->g; p.u = a->u; p.h = h; p.dg = dg; p.du = du;
  set_act(p, a);
  product_gate_grad(p, st);
  // dx = dg gate + du up
  ProductArgs q{};
  q.dtype = q.ctype = a->type;
  q.M = (int)a->rows; q.N = a->width; q.K = a->hidden; q.pairs = 2;
  q.a[0] = {dg, F, 1}; q.b[0] = {a->gate, 1, a->ldgate};
  q.a[1] = {du, F, 1}; q.b[1] = {a->up, 1, a->ldup};
  q.c = a->dx; q.ldc = a->lddx;
  product_store(q, st);
  // the weights' gradients: sums over the rows
  ProductArgs w{};
  w.dtype = w.ctype = a->type;
  w.K = (int)a->rows; w.pairs = 1;
  w.M = a->hidden; w.N = a->width; w.ldc = D;
  w.b[0] = {a->x, 1, a->ldx};
  w.a[0] = {dg, 1, F}; w.c = a->dgate;
  product_store(w, st);
  w.a[0] = {du, 1, F}; w.c = a->dup;
  product_store(w, st);
  w.M = a->width; w.N = a->hidden; w.ldc = F;
  w.a[0] = {a->dy, 1, a->lddy}; w.b[0] = {h, 1, F}; w.c = a->ddown;
  product_store(w, st);
  return m.used;
}

// ---- cross entropy ----
void check_ce(const CrossEntropyArgs* a) {
  require(a, "no arguments");
  check_type(a->type);
  require(a->rows >= 0 && a->rows < MAX_ROWS, "CrossEntropy: bad number of rows");
  require(a->width >= 1 && a->width < MAX_ROWS, "CrossEntropy: bad width");
  require(a->vocab >= 1, "CrossEntropy: bad number of table rows");
}
void check_ce_tensors(const CrossEntropyArgs* a) {
  check_matrix(a->x, a->ldx, a->rows, a->width, "CrossEntropy: x");
  check_matrix(a->table, a->ldtable, a->vocab, a->width, "CrossEntropy: table");
  require(a->target || !a->rows, "CrossEntropy: target");
  require(a->lse || !a->rows, "CrossEntropy: lse");
}

size_t ce_forward(const CrossEntropyArgs* a, void* ws, hipStream_t st) {
  Arena m{(char*)ws};
  const long n = a->rows;
  const int parts = softmax_parts(a->vocab);
  RowsArgs r{a->target, nullptr, n, a->ignore, a->vocab};
  r.rows = m.take<int>(n); r.tgt = m.take<int>(n); r.count = m.take<int>(1);
  r.picked = m.take<float>(n); r.loss = a->loss; r.lse = a->lse;
  void* xc = m.bytes((size_t)n * a->width * dtype_size(a->type));
  float2* part = m.take<float2>((size_t)n * parts);
  if (!ws) return m.used;
  kept_rows(r, st);
  gather_rows(a->x, a->ldx, xc, a->width, r.rows, r.count, n, a->width, a->type, st);
  ProductArgs p{};
  p.dtype = a->type;
  p.M = (int)n; p.N = a->vocab; p.K = a->width; p.pairs = 1;
  p.a[0] = {xc, a->width, 1};
  p.b[0] = {a->table, a->ldtable, 1};
  p.count = r.count; p.target = r.tgt; p.picked = r.picked; p.part = part; p.parts = parts;
  product_softmax(p, st);
  softmax_finish(part, parts, r.picked, r.rows, r.count, n, a->loss, a->lse, st);
  return m.used;
}

// Rows of the table whose gradients of the logits are held at a time: those
// of all rows of x take at most 256 MiB, what the last-level cache holds.
int piece_rows(const CrossEntropyArgs* a) {
  const long most = (256L << 20) / (std::max<long>(a->rows, 1) * dtype_size(a->type));
  return (int)std::min<long>(a->vocab, std::max<long>(1024, most / 1024 * 1024));
}

size_t ce_backward(const CrossEntropyArgs* a, void* ws, hipStream_t st) {
  Arena m{(char*)ws};
  const long n = a->rows, D = a->width;
  const int piece = piece_rows(a);
  RowsArgs r{a->target, a->dloss, n, a->ignore, a->vocab};
  r.rows = m.take<int>(n); r.tgt = m.take<int>(n); r.count = m.take<int>(1);
  if (a->type == DT_F16) r.scale = m.take<float>(1);
  else m.take<float>(1);
  void* xc = m.bytes((size_t)n * D * dtype_size(a->type));
  float* acc = m.take<float>((size_t)n * D);
  void* dl = m.bytes((size_t)n * piece * dtype_size(a->type));
  if (!ws) return m.used;
  kept_rows(r, st);
  gather_rows(a->x, a->ldx, xc, D, r.rows, r.count, n, a->width, a->type, st);
  for (long v0 = 0; v0 < a->vocab; v0 += piece) {
    const int len = (int)std::min<long>(piece, a->vocab - v0);
    const char* rows = (const char*)a->table + v0 * a->ldtable * dtype_size(a->type);
    ProductArgs p{};
    p.dtype = p.ctype = a->type;
    p.pairs = 1; p.count = r.count;
    p.M = (int)n; p.N = len; p.K = a->width;
    p.a[0] = {xc, D, 1};
    p.b[0] = {rows, a->ldtable, 1};
    p.c = dl; p.ldc = piece;
    p.n0 = (int)v0; p.target = r.tgt; p.rows = r.rows; p.lse = a->lse; p.grad = a->dloss; p.scale = r.scale;
    product_softmax_grad(p, st);
    ProductArgs q{};
    q.dtype = a->type; q.ctype = DT_F32;
    q.pairs = 1; q.count = r.count;
    q.M = (int)n; q.N = a->width; q.K = len;
    q.a[0] = {dl, piece, 1};
    q.b[0] = {rows, 1, a->ldtable};
    q.c = acc; q.ldc = D; q.add = v0 > 0;
    product_store(q, st);
    ProductArgs w{};
    w.dtype = w.ctype = a->type;
    w.pairs = 1; w.count = r.count; w.count_k = true;
    w.M = len; w.N = a->width; w.K = (int)n;
    w.a[0] = {dl, 1, piece};
    w.b[0] = {xc, 1, D};
    w.c = (char*)a->dtable + v0 * D * dtype_size(a->type); w.ldc = D;
    w.unscale = r.scale;
    product_store(w, st);
  }
  scatter_rows(acc, D, r.rows, r.count, r.scale, a->dx, a->lddx, n, a->width, a->type, st);
  return m.used;
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
  return sized([&] { check_mlp(a); return mlp_forward(a, nullptr, nullptr); });
}
int GatedMLP(const GatedMLPArgs* a, void* stream) {
  return clr::guarded([&] {
    check_mlp(a);
    check_mlp_tensors(a);
    check_matrix(a->y, a->ldy, a->rows, a->width, "GatedMLP: y");
    require(!a->g == !a->u, "GatedMLP: g and u are kept together");
    if (!a->rows) return;
    check_space(a->workspace, a->workspaceBytes, mlp_forward(a, nullptr, nullptr));
    mlp_forward(a, a->workspace, (hipStream_t)stream);
  });
}
long GatedMLPGradWorkspace(const GatedMLPArgs* a) {
  return sized([&] { check_mlp(a); return mlp_backward(a, nullptr, nullptr); });
}
int GatedMLPGrad(const GatedMLPArgs* a, void* stream) {
  return clr::guarded([&] {
    check_mlp(a);
    check_mlp_tensors(a);
    check_matrix(a->dy, a->lddy, a->rows, a->width, "GatedMLPGrad: dy");
    check_matrix(a->dx, a->lddx, a->rows, a->width, "GatedMLPGrad: dx");
    require((a->g && a->u) || !a->rows, "GatedMLPGrad: g and u");
    require(a->dgate && a->dup && a->ddown, "GatedMLPGrad: the weights' gradients");
    const size_t n = (size_t)a->width * a->hidden * dtype_size(a->type);
    if (!a->rows) {
      for (void* p : {a->dgate, a->dup, a->ddown}) fill_zero(p, n, (hipStream_t)stream);
      return;
    }
    check_space(a->workspace, a->workspaceBytes, mlp_backward(a, nullptr, nullptr));
    mlp_backward(a, a->workspace, (hipStream_t)stream);
  });
}

long CrossEntropyWorkspace(const CrossEntropyArgs* a) {
  return sized([&] { check_ce(a); return ce_forward(a, nullptr, nullptr); });
}
int CrossEntropy(const CrossEntropyArgs* a, void* stream) {
  return clr::guarded([&] {
    check_ce(a);
    check_ce_tensors(a);
    require(a->loss || !a->rows, "CrossEntropy: loss");
    if (!a->rows) return;
    check_space(a->workspace, a->workspaceBytes, ce_forward(a, nullptr, nullptr));
    ce_forward(a, a->workspace, (hipStream_t)stream);
  });
}
long CrossEntropyGradWorkspace(const CrossEntropyArgs* a) {
  return sized([&] { check_ce(a); return ce_backward(a, nullptr, nullptr); });
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
    check_space(a->workspace, a->workspaceBytes, ce_backward(a, nullptr, nullptr));
    ce_backward(a, a->workspace, (hipStream_t)stream);
  });
}

}  // extern "C"
