// paged_rows.h — which sequence a row of a ragged batch belongs to, as the kernels
// that write rows into a paged cache and read them back find it.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace neptune {
namespace {

// floor(x / d), inv = floor((2^32 - 1) / d): the estimate is that or one less
__device__ inline uint32_t divide(uint32_t x, uint32_t d, uint32_t inv) {
  const uint32_t q = __umulhi(x, inv);
  return x - q * d >= d ? q + 1 : q;
}

// The search's first load, for the caller to issue ahead of others: the end of the
// lane's chunk of ceil(B / 64) sequences (cu nullable: there is none to look for).
__device__ inline int chunk_end(const int32_t *cu, int B, int lane) {
  const int chunk = (B + 63) >> 6;
  int end = 0x7fffffff;
  if (cu && lane * chunk < B) end = cu[min((lane + 1) * chunk, B)];
  return end;
}

// The sequence of row tok, the same for LPR lanes together: as many ends of sequences
// lie at or before the row (B: behind the last). Among 64 ends of whole chunks, then
// among those of the chunk that the row is in (1024 single tokens appended 6.9 us, 2048
// 10.6; with a step per 64 sequences 9.7 and 19.3).
template <int LPR>
__device__ inline int sequence_of(const int32_t *cu, int B, int lane, int tok, int end) {
  constexpr int GROUPS = 64 / LPR;
  const int chunk = (B + 63) >> 6;
  int row[GROUPS], at[GROUPS];
  int b = 0;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    row[g] = __builtin_amdgcn_readlane(tok, g * LPR);
    at[g] = chunk * __builtin_popcountll(__ballot(end <= row[g]));
    if (lane / LPR == g) b = at[g];
  }
  if (chunk > 1)
    for (int j = lane; j - lane < chunk; j += 64) {
      int ends[GROUPS];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        ends[g] = j < chunk && at[g] + j < B ? cu[at[g] + j + 1] : 0x7fffffff;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int n = __builtin_popcountll(__ballot(ends[g] <= row[g]));
        if (lane / LPR == g) b += n;
      }
    }
  return b;
}

}  // namespace
}  // namespace neptune
