// Arguments of the tiled kernels of attention with score rules (attend_mfma.h for half widths, attend_parts.h for
// float32, whose buffers are float), of the kernel that finds
// documents' ranges and of the one that mends blocks with non-finite totals (attend_mend.hip).
#pragma once

#include "attend_rules.h"

namespace limn {

constexpr int ATT_ROWS = 128;  // resident rows of a workgroup

struct FastArgs {
  const u16* q;
  const u16* k;
  const u16* v;
  const u16* out;
  const u16* dout;
  const float* lse_in;
  float* delta;
  const int4* ranges;  // (batch, granules): documents of 32 positions, see attend_ranges; nullptr without
  u16* o0;             // out / dq / dk
  u16* o1;             // dv
  float* lse;
  int* odd;            // one flag a block of resident rows: its totals were not all finite
  int64_t batch;
  int heads, kv_heads, hd, granules;
  int head_group;      // see att_head_and_block
  float scale;
  // dK/dV pass of a call with too few key blocks for the GPU: blockIdx.y is a part of the query heads times one of the
  // query tiles, whose float totals go to partial (part, dk and dv, key rows, hd) for attend_join_keys to add
  int head_parts, tile_parts;
  float* partial;
  // backward past 64 half-width dims: the score gradients on their way from the dK/dV pass to the dQ pass, or nullptr:
  // (heads of all sequences, row_blocks, key_tiles, 64 keys, 128 queries)
  u16* ds;
  int row_blocks, key_tiles;
};

int launch_attend_ranges(const RuleArgs& ra, int4* ranges, int64_t batch, int granules, hipStream_t stream);
int launch_attend_delta(const FastArgs& g, int64_t rows, int dtype, hipStream_t stream);
int launch_attend_mend_fwd(const FastArgs& g, const RuleArgs& ra, int dtype, hipStream_t stream);
// blocks of the dQ pass (g.odd) and of the dK/dV pass (kv.odd) that are to be computed again
int launch_attend_mend_bwd(const FastArgs& g, const FastArgs& kv, const RuleArgs& ra, int dtype, hipStream_t stream);
// the packed rows of a forward call whose results are not all finite
int launch_attend_mend_rows(const AttendArgs& a);

#define LIMN_ATTEND_PASSES(D)                                                                              \
  int launch_attend_fwd_##D(const FastArgs& g, const RuleArgs& ra, int dtype, hipStream_t stream);         \
  int launch_attend_dq_##D(const FastArgs& g, const RuleArgs& ra, int dtype, hipStream_t stream);          \
  int launch_attend_dkv_##D(const FastArgs& g, const RuleArgs& ra, int dtype, hipStream_t stream);
LIMN_ATTEND_PASSES(64)
LIMN_ATTEND_PASSES(96)
LIMN_ATTEND_PASSES(128)
int launch_attend_fwd_parts(const FastArgs& g, const RuleArgs& ra, hipStream_t stream);
int launch_attend_dq_parts(const FastArgs& g, const RuleArgs& ra, hipStream_t stream);
int launch_attend_dkv_parts(const FastArgs& g, const RuleArgs& ra, hipStream_t stream);
#undef LIMN_ATTEND_PASSES

}  // namespace limn
