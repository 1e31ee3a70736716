// chunk_index.cpp -- the index arithmetic of kyro_b200/csrc/chunk_index.h for
// a test on the CPU.
#include "chunk_index.h"

extern "C" int hidden_cols(int tok_min, int tok0, int group) {
  return kyro::chunk::hidden_cols(tok_min, tok0, group);
}
extern "C" int chunk_rows(int s0, int s1, int64_t ctx, int T, int max_slots) {
  return kyro::chunk::chunk_rows(s0, s1, ctx, T, max_slots);
}
extern "C" int evict_fits(int64_t len, int reserved, int64_t table_slots, int64_t score_slots) {
  return kyro::chunk::evict_fits(len, reserved, table_slots, score_slots);
}
