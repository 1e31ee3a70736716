// chunk_index.cpp -- the index arithmetic of kyro_b200/csrc/chunk_index.h for
// a test on the CPU.
#include "chunk_index.h"

extern "C" int hidden_cols(int tok_min, int tok0, int group) {
  return kyro::chunk::hidden_cols(tok_min, tok0, group);
}
