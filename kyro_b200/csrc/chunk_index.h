// chunk_index.h -- index arithmetic of the operators on packed prompt chunks
// that has to hold at the limits of what they accept.  It compiles as CUDA
// and as plain C++, so that a test can go through the limits on the CPU.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define KYRO_HD __host__ __device__ __forceinline__
#else
#define KYRO_HD inline
#endif

namespace kyro {
namespace chunk {

// The new tokens of a sequence whose rows are s0 .. s1 - 1 of T and whose
// slots begin at ctx; -1: its rows leave the packed tensors, or its slots the
// max_slots that there is room for.  (ctx is any 64-bit number, so nothing is
// added to it.)
KYRO_HD int chunk_rows(int s0, int s1, int64_t ctx, int T, int max_slots) {
  if (s0 < 0 || s1 < s0 || s1 > T) return -1;
  const int n = s1 - s0;
  return n > 0 && (ctx < 0 || ctx > max_slots - n) ? -1 : n;
}

// Whether a sequence of len slots and `reserved` more fits a table of
// table_slots and the scores' width.
KYRO_HD bool evict_fits(int64_t len, int reserved, int64_t table_slots, int64_t score_slots) {
  return len <= table_slots - reserved && len <= score_slots;
}

// The columns of a step of scores (tokens from tok0 on, `group` heads each)
// that do not see a slot, which tokens from tok_min on see: the first so
// many.  A slot of the context has tok_min = t - ctx, down to -2^30, so the
// difference is cut at zero before it is multiplied; it is no more than the
// slots of an item and the tokens of a step, 256 + 128 / group.
KYRO_HD int hidden_cols(int tok_min, int tok0, int group) {
  const int d = tok_min - tok0;
  return d > 0 ? d * group : 0;
}

}  // namespace chunk
}  // namespace kyro
