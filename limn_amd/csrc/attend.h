// Internal launch interface between the C ABI (attend.hip) and the kernels of attention with score rules.
#pragma once

#include "common.h"

namespace limn {

// One call, already validated. Row r of key head kvh is query i = r / group of head kvh * group + r % group
// (group = heads / kv_heads): a key head's queries are one matrix of group * t_q rows, so grouped heads
// share what is read of k and v, and the gradients of a shared head are one sum in a fixed order.
struct AttendArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* slopes;   // (heads) or nullptr
  const int* documents;  // (batch, t_k) or nullptr
  const int* prefix;     // (batch) or nullptr
  const int* lengths;    // (batch) or nullptr
  const void* out;       // backward
  const float* lse;      // backward
  const void* dout;      // backward
  void* o0;              // out / dq
  void* o1;              // lse / dk
  void* o2;              // dv
  int dtype;
  int64_t batch, heads, kv_heads, t_q, t_k, hd, hd_v;
  bool causal;
  double scale, softcap;
  void* workspace;
  int64_t workspace_bytes;
  hipStream_t stream;
  int64_t group() const { return heads / kv_heads; }
};

// Kernels in float arithmetic for every type and head dim up to 256 (attend_general.h).
int64_t attend_general_workspace(const AttendArgs& a, bool backward);
int launch_attend_general_fwd(const AttendArgs& a);
int launch_attend_general_bwd(const AttendArgs& a);

// Joins `splits` partial results of `rows` packed rows: totals (splits, rows, hd_v) float, and stats
// (splits, rows, 2) float (reference point of the exponentials in log2, sum), into out and lse; sums and totals
// are 2^up times the weights'. A split that has seen nothing is not read.
int launch_attend_join(const AttendArgs& a, const float* totals, const float* stats, int64_t splits, float up);

// Few queries against a cache, half widths (attend_token.hip).
int64_t attend_token_workspace(const AttendArgs& a);
int launch_attend_token(const AttendArgs& a);

// bytes rounded up to where the next part of a workspace may start
constexpr int64_t attend_align(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace limn
