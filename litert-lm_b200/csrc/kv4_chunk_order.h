// Which barrier, and which of its phases, every wait of the chunk kernel (kv4_attn_tc.cuh) is for.  Kept apart from the kernel so that
// the orders in which its threads can meet them are walked through on the host.
//
// A wait names a phase by its parity only, so it tells phase c from c - 2 by what the waiting thread has seen before: it must know
// that phase c - 1 is over.  The issuing warp and the softmax warps know where they are; what the softmax warps do not see
// is every O.  S(j) says that O(j - 2) is complete (the issuer waited for it), so the wait for O(j - 1) in the loop is sound, but after
// the last tile they know of O(n - 3) only: the end has a barrier of its own that completes once.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define B2_CHUNK_FN __host__ __device__ __forceinline__ constexpr
#else
#define B2_CHUNK_FN inline constexpr
#endif

namespace b200lm {

// Words of the barriers: one a stage (tile j uses stage j & 1), or one alone.
enum KcBar : int { kKcKFull = 0, kKcKEmpty = 2, kKcVFull = 4, kKcVEmpty = 6, kKcSFull = 8, kKcPFull = 10, kKcOFull = 12, kKcQReady = 13, kKcODone = 14, kKcBars = 15 };

struct KcWait {
  int bar;
  int phase;                                               // phases of a barrier count from 0
  B2_CHUNK_FN uint32_t parity() const { return (uint32_t)(phase & 1); }
};
B2_CHUNK_FN int kc_stage(int bar, int j) { return bar + (j & 1); }
// K or V of tile j, scores of tile j, probabilities of tile j.
B2_CHUNK_FN KcWait kc_full(int bar, int j) { return {kc_stage(bar, j), j >> 1}; }
// The stage of tile j (j >= 2) read by the products of tile j - 2.
B2_CHUNK_FN KcWait kc_empty(int bar, int j) { return {kc_stage(bar, j), (j >> 1) - 1}; }
// O of tile j, for those who know that O of tile j - 1 is complete.
B2_CHUNK_FN KcWait kc_o(int j) { return {kKcOFull, j}; }
// All products.
B2_CHUNK_FN KcWait kc_end() { return {kKcODone, 0}; }

}  // namespace b200lm
