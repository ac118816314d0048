// preference.h -- launches of preference.hip.
#pragma once
#include "cleartext.h"

enum PairLoss { PAIR_LOGISTIC = 0, PAIR_HINGE = 1 };

// Sequence s of 2 * pairs has the tokens offsets[s] .. offsets[s + 1] of a line
// of `length`, or without offsets a row of `length` of each matrix.
struct PairArgs {
  const float* loss; long ldloss;
  const float* reference; long ldreference;   // may be null: 0
  const long long* target; long ldtarget;     // may be null: every token counts
  const long long* offsets;
  float* value; float* ratio; float* slope;   // [pairs], [pairs][2], [pairs][2]
  long long* kept;                            // [pairs]: whether a token of the pair counts; may be null
  const float* dvalue;                        // backward
  float* dloss; long lddloss;
  void* workspace;
  long pairs, length;
  long long ignore;
  int kind; bool average;
  float beta, margin, smoothing;
  int splits;                                 // (of the launch)
};
size_t preference_workspace(long pairs, long length, bool packed);
void preference_launch(PairArgs a, hipStream_t st);
void preference_grad_launch(PairArgs a, hipStream_t st);
