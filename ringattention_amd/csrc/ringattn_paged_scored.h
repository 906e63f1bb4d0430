// gfx950 (CDNA4) kernel: attention of new tokens over a paged cache with scores that are capped, biased by distance, or masked by documents and
// prefixes (the programs of ringattn_paged_few.h and ringattn_paged_many.h; ringattn_paged_attend.hip has those of plain scores).
//
// A file for each dim (ringattn_paged_scored.hip, ringattn_paged_scored64.hip), which compile beside each other.
//
//   paged_scored_kernel : SC says what becomes of a score between the products and the softmax (shape_scores), in registers, where the
//       vector pipes have what the matrix cores leave them: a cap is an exponential and a reciprocal more, a slope an addition and a fused
//       multiply-add.  Masks cost what those of a window cost: only tiles that some row of a wave may not see are compared.
#pragma once
#include "ringattn_paged_few.h"
#include "ringattn_paged_many.h"

namespace ringattn {
namespace paged {

template <int DT, int D, int SC>
__global__ __launch_bounds__(512, 2) void paged_scored_kernel(const AttendArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kFewLds<D> > kManyLds<D> ? kFewLds<D> : kManyLds<D>];
  const int few = (int)blockIdx.x - a.few_begin;
  if ((unsigned)few < (unsigned)kFewWorkgroups) few_rows<DT, D, SC>(a, smem, few);
  else many_rows<DT, D, SC>(a, smem, few < 0 ? (int)blockIdx.x : few - kFewWorkgroups);
}

// Of calls that can have few rows only, single tokens above all: the code of many rows is not between theirs, which is fetched as it runs.  (A token over
// 512, 8 heads x 64, capped: 9.7 us in the kernel of both, 8.7 here; 48 single tokens over some 3 K, 16/4 heads x 128 75.5 and 74.6.)
template <int DT, int D, int SC> __global__ __launch_bounds__(512, 2) void paged_scored_few_kernel(const AttendArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kFewLds<D>];
  few_rows<DT, D, SC>(a, smem, (int)blockIdx.x);
}

// As paged_merge_kernel: which row tiles were cut goes by the prefixes too.
template <int DT, int D> __global__ __launch_bounds__(64 * kMergeSharers) void paged_scored_merge_kernel(const AttendArgs a) {
  __shared__ float sums[2][kMergeSharers - 1][18][64];
  for (int64_t block = blockIdx.x, turn = 0; block < INT32_MAX && merge_many<DT, D, kScored>(a, (int)block, sums[turn]); block += gridDim.x, turn ^= 1) {}
}

template <int DT, int D> static hipError_t launch_scored(const AttendArgs& a, int sc, int64_t many_places, int64_t cut_tiles, hipStream_t stream) {
  const int64_t blocks = kFewWorkgroups + many_places * a.kv_heads, merges = a.many_cut ? cut_tiles * a.kv_heads * (kManyRows / 32) * (D / 32) : 0;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
#define RA_LAUNCH(SC_)                                                                                              \
  case SC_:                                                                                                        \
    if (many_places == 0) paged_scored_few_kernel<DT, D, SC_><<<kFewWorkgroups, 512, 0, stream>>>(a);               \
    else paged_scored_kernel<DT, D, SC_><<<(unsigned)blocks, 512, 0, stream>>>(a);                                  \
    break
  switch (sc) {
    RA_LAUNCH(kScored);
    RA_LAUNCH(kScored | kCapped);
    RA_LAUNCH(kScored | kSloped);
    RA_LAUNCH(kScored | kCapped | kSloped);
    default: return hipErrorInvalidValue;
  }
#undef RA_LAUNCH
  if (merges > 0) paged_scored_merge_kernel<DT, D><<<(unsigned)(merges < 1024 ? merges : 1024), 64 * kMergeSharers, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace ringattn
