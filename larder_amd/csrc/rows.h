// What the kernels of the trunk's attention share (rope.hip, attend.hip, prompt.hip): the place of a packed row in its
// sequence, the cos / sin of a position, matrix-core fragments.
#pragma once
#include "grouped.h"

namespace lmoe {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Workgroups of 256 a launch may have: the runtime cuts a grid of 2^32 threads or more without a word
constexpr long long kMostGroups = (1ll << 24) - 1;

// The largest b < B with first(cu[b], b) <= t, by one wavefront (-1 if there is none); first never falls with b where cu
// does not. A load for every factor of 64 in B. Whatever cu holds, the result is in [-1, B); where cu falls, t may lie before what
// that b begins with, which callers look at before they take it for an index.
template <typename F>
__device__ __forceinline__ int last_at(const int *cu, int B, int t, F &&first) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = B;  // how many b there are is in [lo, hi]
  while (hi - lo > 64) {
    const int step = (hi - lo + 63) >> 6, i = lo + (lane + 1) * step - 1;
    lo += step * __popcll(__ballot(i < hi && first(cu[min(i, hi - 1)], i) <= (long long)t));
    hi = min(lo + step, hi);
  }
  if (lo < hi) {
    const int b = min(lo + lane, hi - 1);
    lo += __popcll(__ballot(lo + lane < hi && first(cu[b], b) <= (long long)t));
  }
  return __builtin_amdgcn_readfirstlane(lo - 1);
}

// A sequence's rows [row0, row0 + n) of T packed ones: cu[b] .. cu[b + 1], or row b alone where cu is null. Offsets past
// the rows that there are (or that fall) leave an empty sequence, never a row out of bounds. Where offsets fall (false), other
// sequences may have the same rows.
__device__ __forceinline__ bool seq_rows(const int *cu, int b, int T, int *row0, int *n) {
  if (!cu) {
    *row0 = b;
    *n = b < T ? 1 : 0;
    return true;
  }
  const int a = cu[b], next = cu[b + 1], e = min(next, T);
  *row0 = a;
  *n = a < 0 || e <= a ? 0 : e - a;
  return next >= a;
}

}  // namespace lmoe
