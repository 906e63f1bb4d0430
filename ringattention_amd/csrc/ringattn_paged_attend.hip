// gfx950 (CDNA4) kernel: attention of new tokens over a paged cache (ringattn_paged_few.h and ringattn_paged_many.h hold the programs).
//
//   paged_attend_kernel : one launch for a whole batch.  256 of its workgroups have the sequences of few query rows, a run of key tiles
//       each; the others those of many, 256 rows each.  A batch may have both -- a chunk of one prompt beside the next tokens of other
//       sequences --, and which sequences have how many rows only the device knows: also of a sequence alone, whose new tokens may be
//       fewer than the rows of q.
#include "ringattn_paged_few.h"
#include "ringattn_paged_many.h"

namespace ringattn {
namespace paged {

template <int DT, int D>
__global__ __launch_bounds__(512, 2) void paged_attend_kernel(const AttendArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kFewLds<D> > kManyLds<D> ? kFewLds<D> : kManyLds<D>];
  const int few = (int)blockIdx.x - a.few_begin;
  if ((unsigned)few < (unsigned)kFewWorkgroups) few_rows<DT, D>(a, smem, few);
  else many_rows<DT, D>(a, smem, few < 0 ? (int)blockIdx.x : few - kFewWorkgroups);
}

// As many workgroups as are at work at a time: how many row tiles were cut only the device knows.
template <int DT, int D> __global__ __launch_bounds__(64 * kMergeSharers) void paged_merge_kernel(const AttendArgs a) {
  // In turn, so that one barrier each suffices: what one call of merge_many reads behind its barrier, the call after the next writes in front
  // of its own, and between the two lies that of the next.
  __shared__ float sums[2][kMergeSharers - 1][18][64];
  for (int64_t block = blockIdx.x, turn = 0; block < INT32_MAX && merge_many<DT, D>(a, (int)block, sums[turn]); block += gridDim.x, turn ^= 1) {}
}

hipError_t launch_paged_attend(const AttendArgs& a, int dtype, int dim, int64_t many_places, int64_t cut_tiles, hipStream_t stream) {
  const int64_t blocks = kFewWorkgroups + many_places * a.kv_heads, merges = a.many_cut ? cut_tiles * a.kv_heads * (kManyRows / 32) * (dim / 32) : 0;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
#define RA_LAUNCH_ATTEND(DT_, D_)                                                                             \
  do {                                                                                                       \
    paged_attend_kernel<DT_, D_><<<(unsigned)blocks, 512, 0, stream>>>(a);                                    \
    if (merges > 0) paged_merge_kernel<DT_, D_><<<(unsigned)(merges < 1024 ? merges : 1024), 64 * kMergeSharers, 0, stream>>>(a);                  \
  } while (0)
  if (dtype == 0 && dim == 64) RA_LAUNCH_ATTEND(0, 64);
  else if (dtype == 1 && dim == 64) RA_LAUNCH_ATTEND(1, 64);
  else if (dtype == 0 && dim == 128) RA_LAUNCH_ATTEND(0, 128);
  else if (dtype == 1 && dim == 128) RA_LAUNCH_ATTEND(1, 128);
#undef RA_LAUNCH_ATTEND
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace paged
}  // namespace ringattn
