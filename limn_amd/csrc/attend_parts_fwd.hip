// One pass of attend_parts.h.
#include "attend_parts.h"

namespace limn {
int launch_attend_fwd_parts(const FastArgs& g, const RuleArgs& ra, hipStream_t stream) { return launch_parts<ATTEND_PASS_FWD>(g, ra, stream); }
}  // namespace limn
