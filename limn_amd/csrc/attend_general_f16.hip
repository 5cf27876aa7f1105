// attend_general.h for float16 storage.
#include "attend_general_launch.h"

namespace limn {
int attend_general_fwd_f16(const AttendArgs& a, int64_t splits) { return gen_fwd<F16>(a, splits); }
int attend_general_bwd_f16(const AttendArgs& a) { return gen_bwd<F16>(a); }
}  // namespace limn
