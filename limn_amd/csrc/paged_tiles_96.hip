// paged_tiles.h at one tile width.
#include "paged_tiles.h"

namespace limn {
int launch_paged_tiles_96(const PagedArgs& a, const PagedFast& f) {
  return a.dtype == LIMN_HIP_BFLOAT16 ? launch_tiles_rules<BF16, 96>(a, f) : launch_tiles_rules<F16, 96>(a, f);
}
}  // namespace limn
