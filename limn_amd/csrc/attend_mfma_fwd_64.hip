// One pass of attend_mfma.h at one tile width.
#include "attend_mfma.h"

namespace limn {
int launch_attend_fwd_64(const FastArgs& g, const RuleArgs& ra, int dtype, hipStream_t stream) {
  return dtype == LIMN_HIP_BFLOAT16 ? launch_fast_rules<ATTEND_PASS_FWD, BF16, 64>(g, ra, stream) : launch_fast_rules<ATTEND_PASS_FWD, F16, 64>(g, ra, stream);
}
}  // namespace limn
