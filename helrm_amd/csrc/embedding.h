// embedding.h -- launches of embedding.hip.
#pragma once
#include "cleartext.h"

struct EmbedArgs {
  const long long* ids;             // [tokens]
  const void* table; long ldtable;  // [vocab][width]
  void* y; long ldy;                // forward: the rows; backward: their gradient
  void* dtable;                     // [vocab][width]
  void* workspace;
  long tokens; int width, vocab, dtype;
  long long ignore;
  float scale;
};
void embedding_launch(const EmbedArgs& a, hipStream_t st);
size_t embedding_grad_workspace(long tokens, int width, int vocab, int dtype);
void embedding_grad_launch(const EmbedArgs& a, hipStream_t st);
