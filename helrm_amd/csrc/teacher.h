// teacher.h -- launches of teacher.hip: what a distillation does beside the
// products of products.hip and skinny.hip.
#pragma once
#include "cleartext.h"

constexpr int MOST_TOP = 1024;   // a teacher's logits of a row

// Of each row, its entries (ids other than `ignore`, logits above -inf):
// scores[j] = <x, table[ids[j]]> / temperature, probs[j] the softmax of logits
// / temperature, of an id that is there again with the first one; -1 of
// what is no entry, or again.  kept: 0 of a row without entries, 2 of one with an
// id outside [0, vocab) (NaN in both), else 1.
struct TeachArgs {
  const void* x; long ldx;
  const void* table; long ldtable;
  const long long* ids; const void* logits;   // [rows][top]
  float* scores; float* probs;
  long long* kept;                            // [rows]
  long rows; int width, vocab, top, dtype, teacher_type;
  long long ignore;
  float temperature;
  int parts;                                  // (of the launch)
};
constexpr int TEACH_NONE = 0, TEACH_FINE = 1, TEACH_OUTSIDE = 2;
void teach_entries(TeachArgs a, hipStream_t st);

// The pieces of each row's softmax joined: lse, and loss = temperature^2 times
// the divergence of the teacher's distribution from the softmax.
struct TeachFinish {
  const float2* part; int parts;              // [rows that count][parts]
  const int* rows; const int* count;          // those rows, or null: all, whose loss is 0 where `kept` says so
  const float* scores; const float* probs; const long long* kept;
  float* loss; float* lse;
  long n; int top;
  float temperature;
};
void teach_finish(const TeachFinish& a, hipStream_t st);

// The teacher's part of the logits' gradient, in columns v0 .. v0 + len of dl
// (products.h's layout of a factor): (exp(score - lse) - prob) grad.
struct TeachPatch {
  uint16_t* dl; long ld, part;
  const int* rows; const int* tgt; const int* count;   // of the rows that count
  const float* lse; const float* grad; const float* scale;
  const long long* ids; const float* scores; const float* probs;
  long n; int top, dtype;
  long v0; int len;
};
void teach_patch(const TeachPatch& a, hipStream_t st);
