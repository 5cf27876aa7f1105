// attend_general.h for float32 storage.
#include "attend_general_launch.h"

namespace limn {
int attend_general_fwd_f32(const AttendArgs& a, int64_t splits) { return gen_fwd<F32>(a, splits); }
int attend_general_bwd_f32(const AttendArgs& a) { return gen_bwd<F32>(a); }
}  // namespace limn
