// teacher.h -- launches of teacher.hip: what a distillation does beside the
// products of products.hip and skinny.hip.
#pragma once
#include <algorithm>
#include "cleartext.h"

constexpr int MOST_TOP = 1024;   // a teacher's logits of a row

// Of each row, its entries (ids other than `ignore`, logits above -inf):
// cols[j] the table's row, probs[j] the softmax of logits / temperature, of an id
// that is there again with the first one, scores[j] = <x, table[cols[j]]> /
// temperature.  Places that are no entry have -1 in cols and probs; NaN in
// probs of an id outside [0, vocab).
struct TeachArgs {
  const void* x; long ldx;
  const void* table; long ldtable;
  const long long* ids; const void* logits;   // [rows][top]
  float* scores; float* probs; int* cols;     // [rows][top]
  long long* kept;                            // [rows]: 0 of a row without entries, 2 of one with an id outside, else 1
  long rows; int width, vocab, top, dtype, teacher_type;
  long long ignore;
  float temperature;
  int parts;                                  // workgroups a row, of a launch that computes scores (entry_parts)
  // teach_order: rows that count, and where its entries of each tile of 2^shift columns begin
  const int* which; const int* count;
  uint16_t* starts; int tiles, shift;         // [rows][tiles + 1]
};
constexpr int TEACH_NONE = 0, TEACH_FINE = 1, TEACH_OUTSIDE = 2;
// 512 workgroups, if there are as many times the 16 entries that the smallest one takes at once
inline int entry_parts(long rows, int top) { return (int)std::max(1L, std::min((511 + rows) / rows, (top + 15L) / 16)); }
inline size_t entries_bytes(int top) { return (size_t)((top + 3) & ~3) * 8 + 16 * 4; }   // of LDS
void teach_entries(const TeachArgs& a, hipStream_t st);
// The same in two steps, in the order of cols, for scores that a product picks out: kept; the rest but scores.
void teach_kept(const TeachArgs& a, hipStream_t st);
void teach_order(const TeachArgs& a, hipStream_t st);

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
  const int* cols; const float* scores; const float* probs;
  long n; int top, dtype;
  long v0; int len;
};
void teach_patch(const TeachPatch& a, hipStream_t st);
