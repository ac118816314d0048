// skinny.h -- launches of skinny.hip.
#pragma once
#include "cleartext.h"

inline long skinny_rows(int dtype) { return dtype == DT_F32 ? 64 : 16; }   // the most rows of X

struct SkinnyArgs {
  const void* x; long ldx;           // [T][K]; float32 for skinny_store
  const void* w; long ldw;           // [N][K]
  const void* w2; long ldw2;         // gate: the up projection
  int T, N, K, dtype;                // of x, w and out; any alignment
  void* out; long ldout;             // [T][N]; float32 of skinny_gate
  float* g; float* u; long ldg;      // gate: [T][ldg] kept projections, 0 past N; may be null
  int act; float coef[4];
  const long long* target; float* picked; float2* part;   // softmax: [T], [T], [T][parts]
  int parts, groups; bool alone;     // (of the launch)
};
// out = act(X W^T) * (X W2^T)
void skinny_gate(SkinnyArgs p, hipStream_t st);
// out = X W^T
void skinny_store(SkinnyArgs p, hipStream_t st);
// loss and lse of every row of X against the rows of W
int skinny_softmax_parts(int N);
void skinny_softmax(SkinnyArgs p, long long ignore, float* loss, float* lse, hipStream_t st);
