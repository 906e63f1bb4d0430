// gfx950 (CDNA4): attention with shaped scores over a paged cache, dim 64 (ringattn_paged_scored.h).
#include "ringattn_paged_scored.h"

namespace ringattn {
namespace paged {

hipError_t launch_paged_scored64(const AttendArgs& a, int sc, int dtype, int64_t many_places, int64_t cut_tiles, hipStream_t stream) {
  if (dtype == 0) return launch_scored<0, 64>(a, sc, many_places, cut_tiles, stream);
  return launch_scored<1, 64>(a, sc, many_places, cut_tiles, stream);
}

}  // namespace paged
}  // namespace ringattn
