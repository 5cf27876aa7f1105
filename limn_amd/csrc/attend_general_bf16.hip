// attend_general.h for bfloat16 storage.
#include "attend_general_launch.h"

namespace limn {
int attend_general_fwd_bf16(const AttendArgs& a, int64_t splits) { return gen_fwd<BF16>(a, splits); }
int attend_general_bwd_bf16(const AttendArgs& a) { return gen_bwd<BF16>(a); }
}  // namespace limn
