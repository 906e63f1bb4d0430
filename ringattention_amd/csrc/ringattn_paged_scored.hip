// gfx950 (CDNA4): attention with shaped scores over a paged cache, dim 128 (ringattn_paged_scored.h).
#include "ringattn_paged_scored.h"

namespace ringattn {
namespace paged {

hipError_t launch_paged_scored64(const AttendArgs& a, int sc, int dtype, int64_t many_places, int64_t cut_tiles, hipStream_t stream);

hipError_t launch_paged_scored(const AttendArgs& a, int sc, int dtype, int dim, int64_t many_places, int64_t cut_tiles, hipStream_t stream) {
  if (dim == 64) return launch_paged_scored64(a, sc, dtype, many_places, cut_tiles, stream);
  if (dtype == 0) return launch_scored<0, 128>(a, sc, many_places, cut_tiles, stream);
  return launch_scored<1, 128>(a, sc, many_places, cut_tiles, stream);
}

}  // namespace paged
}  // namespace ringattn
