// products.h -- launches of products.hip: the matrix products of the gated
// block and of the cross entropy, with what follows each done on the tile.
#pragma once
#include "cleartext.h"

// act(g): silu g/(1 + e^-g), gelu g Phi(g), cubic ((c3 g + c2) g + c1) g + c0
enum Act { ACT_SILU = 0, ACT_GELU = 1, ACT_CUBIC = 2 };

// C[m][n] = sum over k of A(m, k) B(n, k), for one or two pairs of factors
// that are added.  A factor's element (row, k) is at row * s + k * t.
struct Factor { const void* p; long s, t; };

struct ProductArgs {
  Factor a[2], b[2];
  int pairs;
  int M, N, K;
  int dtype;                 // of the factors
  const int* count;          // on the device, may be null: the rows present, in the place of M
  bool count_k;              // in the place of K
  // store
  void* c; long ldc; int ctype; bool add;  // add: c (float32) += the product
  const float* unscale;      // the product is divided by this, where there is one
  // gate
  float* g; float* u;        // [M][N] float32, kept for the backward pass; may be null
  void* h; void* dg; void* du;  // [M][N] in the type of the factors
  int act; float coef[4];
  // softmax: table rows n0 .. n0 + N
  int n0;
  const int* target;         // of tile row i; -1: none (its loss is NaN)
  float2* part; int parts;   // [M][parts] running maximum and sum of a piece of a row
  float* picked;             // the target's logit
  const int* rows;           // row i of the tiles is row rows[i] of lse and grad
  const float* lse; const float* grad;
  const float* scale;        // the gradient's factor in a 16-bit type
};

// h = act(A B0^T) * (A B1^T)
void product_gate(const ProductArgs& p, hipStream_t st);
// dh = A B; dg = dh u act'(g), du = dh act(g), h = act(g) u
void product_gate_grad(const ProductArgs& p, hipStream_t st);
void product_store(const ProductArgs& p, hipStream_t st);
// the products of rows of A with rows of the table go into part and picked
void product_softmax(const ProductArgs& p, hipStream_t st);
// (exp(A B^T - lse) - onehot(target)) grad into c
void product_softmax_grad(const ProductArgs& p, hipStream_t st);
// pieces of a row that product_softmax leaves for a table of N rows
int softmax_parts(int N);

// Rows whose target is not `ignore`, in order: rows[], target[] (-1: outside
// [0, vocab)), *count, and picked[] = NaN; loss and lse (may be null) of the
// others are 0.  scale (may be null): the power of two that brings the
// largest |grad| of these rows near 2^14.
struct RowsArgs {
  const long long* target; const float* grad;
  long n; long long ignore; int vocab;
  int* rows; int* tgt; int* count;
  float* picked; float* loss; float* lse; float* scale;
};
void kept_rows(const RowsArgs& a, hipStream_t st);
// to[i] = from[rows[i]], i < *count
void gather_rows(const void* from, long ld, void* to, long ldto, const int* rows, const int* count, long n, int width, int dtype, hipStream_t st);
// loss[row] = lse - picked, lse = the logarithm of the parts' sum
void softmax_finish(const float2* part, int parts, const float* picked, const int* rows, const int* count, long n, float* loss, float* lse, hipStream_t st);
// out[row] = acc[i] / *scale, 0 for rows that are not kept
void scatter_rows(const float* acc, long ldacc, const int* rows, const int* count, const float* scale, void* out, long ldout, long n, int width, int dtype,
                  hipStream_t st);
void fill_zero(void* p, size_t bytes, hipStream_t st);  // bytes: a multiple of 2
