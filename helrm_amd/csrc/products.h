// products.h -- launches of products.hip: the matrix products of the gated
// block and of the cross entropy, with what follows each done on the tile.
#pragma once
#include <initializer_list>
#include "cleartext.h"
#include "plan.h"

// act(g): silu g/(1 + e^-g), gelu g Phi(g), cubic ((c3 g + c2) g + c1) g + c0
enum Act { ACT_SILU = 0, ACT_GELU = 1, ACT_CUBIC = 2 };

// C[m][n] = sum over k of A(m, k) B(n, k), for up to 12 pairs of factors that
// are added, of which the first `corrections` are settled (tiles.h) before the
// others.  Factors are 16-bit, 16-byte aligned, their rows `ld` elements
// (a multiple of 8) apart and filled up with zeros to a multiple of 8
// elements.  Whether a factor's rows run along k or along m (n) goes by the
// product.
struct ProductArgs {
  const uint16_t* a[12]; const uint16_t* b[12];
  const uint16_t* b2[6];     // gate: the up projection's
  int pairs, corrections;
  long lda, ldb;
  int M, N, K;
  int dtype;                 // of the operator; the factors of a float32 one are its bfloat16 parts
  const int* count;          // on the device, may be null: the rows present, in the place of M
  bool count_k;              // in the place of K
  float* partial;            // product_scratch bytes (but softmax)
  int most = clr::SPLITS;    // splits of k
  int splits;                // (of the launch)
  // store
  void* c; long ldc; int ctype; bool add;  // add: c (float32) += the product
  const float* unscale;      // the product is divided by this, where there is one
  // gate
  float* g; float* u;        // [M][ldh] float32, kept for the backward pass; may be null
  void* h; void* dg; void* du;  // [M][ldh], `hpart` elements from one part to the next (0: one part)
  long ldh, hpart;           // (hpart also of the c of softmax_grad)
  int act; float coef[4];
  // softmax: table rows n0 .. n0 + N
  int n0;
  const int* target;         // of row i of the tiles; -1: none (its loss is NaN)
  float2* part; int parts;   // [M][parts] running maximum and sum of a piece of a row
  float* picked;             // the target's logit
  const float* lse; const float* grad;  // of row i of the tiles
  const float* scale;        // the gradient's factor in a 16-bit type
  float rate;                // teach: of the logits, 1 / temperature
  // (may be null) the columns of each row whose logits are wanted, in order: those of row m in tile n are number
  // starts[m][n] .. starts[m][n + 1] of cols[rows[m]][top], whose logits go to scores
  const uint16_t* starts; long ldstarts;
  const int* rows; const int* cols; float* scores; int top;
};

// h = act(A B^T) * (A B2^T); rows of all three run along k
void product_gate(const ProductArgs& p, hipStream_t st);
// v = A B, A's rows along k, B's along n: dg = v u act'(g), du = v act(g), h = act(g) u
void product_gate_grad(const ProductArgs& p, hipStream_t st);
// Bytes that a product (softmax but) of these shapes needs at `partial`, or products in one launch together.
using clr::Shape;
size_t product_scratch(std::initializer_list<Shape> shapes, long K, int pairs, bool gate = false, int most = clr::SPLITS);
void product_nt(const ProductArgs& p, hipStream_t st);  // A B^T
void product_nn(const ProductArgs& p, hipStream_t st);  // A B
void product_tn(const ProductArgs& p, hipStream_t st);  // A^T B
void product_tn(ProductArgs a, ProductArgs b, ProductArgs c, hipStream_t st);  // three of the same K in one launch, a.partial of all
// the products of rows of A with the N rows of the table go into part, plan.parts pieces a row, and picked
void product_softmax(const ProductArgs& p, const clr::SoftmaxPlan& plan, hipStream_t st);
// (exp(A B^T - lse) - onehot(target)) grad into c, in the layout of a factor
void product_softmax_grad(const ProductArgs& p, hipStream_t st);
// the same of rate A B^T, without a target's part in either (a row whose target is negative has NaN all over)
void product_teach(const ProductArgs& p, const clr::SoftmaxPlan& plan, hipStream_t st);
void product_teach_grad(const ProductArgs& p, hipStream_t st);

// Matrices into the layout above, up to 8 in one launch: row rows[i] (or i) of
// `from` to row i of `to`, for i < *count (or n); a float32 one as three parts
// `part` elements apart.
struct LayOut {
  const void* from; long ld;
  void* to; long ldto, part;
  const int* rows; const int* count;
  long n; int width;
};
void lay_out(const LayOut* jobs, int n, int dtype, hipStream_t st);

// Rows whose target is not `ignore`, in order: rows[], tgt[] (-1: outside [0,
// vocab)), *count.  Forward (loss): picked[] = NaN, and loss and lse of the
// others are 0.  Backward (lse_kept): their lse and grad, and in scale (may be
// null) the power of two that brings the largest |grad| near 2^14.
struct RowsArgs {
  const long long* target; const float* grad;
  long n; long long ignore; int vocab;
  int* rows; int* tgt; int* count;   // of the rows that count: each one's row, its target (-1 outside the table), and how many they are
  int* place;                        // of each row: where it is among them, or -1
  float* picked; float* loss; float* lse; float* lse_kept; float* grad_kept; float* scale;
  float factor = 1.0f;               // of grad, in grad_kept
};
void kept_rows(const RowsArgs& a, hipStream_t st);
// loss[row] = lse - picked, lse = the logarithm of the parts' sum
void softmax_finish(const float2* part, int parts, const float* picked, const int* rows, const int* count, long n, float* loss, float* lse, hipStream_t st);
// out[row] = (acc[place[row]], and what is `second` elements behind it) / *scale, 0 for rows that are not kept
void scatter_rows(const float* acc, long ldacc, long second, const int* place, const float* scale, void* out, long ldout, long n, int width, int dtype,
                  hipStream_t st);
// total[0] = the sum of n losses, or (target) their mean over the rows whose target is not `ignore`; factor[0] = 1, or one over their number
size_t loss_total_bytes(long n);
void loss_total(const float* loss, const long long* target, long long ignore, long n, void* workspace, float* total, float* factor, hipStream_t st);
void fill_zero(void* p, size_t bytes, hipStream_t st);  // bytes: a multiple of 2
