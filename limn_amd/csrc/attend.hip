// The C ABI of attention with score rules (include/limn_hip.h): argument checks, choice of kernels, workspaces;
// and the kernel that joins partial results of a call whose keys are split over workgroups.

#include <math.h>

#include "attend_fast.h"

namespace limn {

int attend_general_fwd_f32(const AttendArgs& a, int64_t splits);
int attend_general_fwd_f16(const AttendArgs& a, int64_t splits);
int attend_general_fwd_bf16(const AttendArgs& a, int64_t splits);
int attend_general_bwd_f32(const AttendArgs& a);
int attend_general_bwd_f16(const AttendArgs& a);
int attend_general_bwd_bf16(const AttendArgs& a);

namespace {

constexpr int JOIN_MOST = 1024;  // splits of a call: both planners stay at or below

// A workgroup per packed row: the splits' reference points brought to the largest, their sums and totals added
// in a fixed order (each wave a run of splits, then the waves), so that the result does not depend on which
// workgroup ended first. A split that saw nothing (no reference point, and a sum of 0: it is NaN where a score
// was) is not read. The factors are found first, a split a thread, so that the loads of the totals do not
// wait for one another: 60 splits of 64 rows took 60 us with one wave that walked them in turn, 5 so.
template <typename T>
__global__ __launch_bounds__(256) void attend_join(const float* __restrict__ totals, const float* __restrict__ stats,
                                                   typename T::Storage* __restrict__ out, float* __restrict__ lse, int64_t rows_all,
                                                   int splits, int group, int t_q, int hd_v, float up) {
  __shared__ float factor[JOIN_MOST], part[4][256], sums[256];
  const int64_t row = blockIdx.x;
  const int64_t per = (int64_t)group * t_q, bk = row / per, r = row % per;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float top = -__builtin_inff();
  for (int s = threadIdx.x; s < splits; s += 256) top = fmaxf(top, stats[(s * rows_all + row) * 2]);
  sums[threadIdx.x] = top;
  __syncthreads();
  for (int h = 128; h > 0; h >>= 1) {
    if (threadIdx.x < h) sums[threadIdx.x] = fmaxf(sums[threadIdx.x], sums[threadIdx.x + h]);
    __syncthreads();
  }
  top = sums[0];
  __syncthreads();
  const float base = top == -__builtin_inff() ? 0.f : top;
  float total = 0.f;
  for (int s = threadIdx.x; s < splits; s += 256) {
    const float m = stats[(s * rows_all + row) * 2], l = stats[(s * rows_all + row) * 2 + 1];
    const float f = m == -__builtin_inff() ? (l == 0.f ? 0.f : 1.f) : fast_exp2(m - base);
    factor[s] = m == -__builtin_inff() && l == 0.f ? -1.f : f;  // -1: not read
    total += l * f;
  }
  sums[threadIdx.x] = total;
  __syncthreads();
  for (int h = 128; h > 0; h >>= 1) {
    if (threadIdx.x < h) sums[threadIdx.x] += sums[threadIdx.x + h];
    __syncthreads();
  }
  total = sums[0];
  const int run = (splits + 3) / 4, s1 = min(splits, (wave + 1) * run);
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const int d = c * 64 + lane;
    float x = 0.f;
    if (d < hd_v) {
#pragma unroll 8
      for (int s = wave * run; s < s1; s++) {
        const float f = factor[s];
        x += f < 0.f ? 0.f : f * totals[(s * rows_all + row) * hd_v + d];
      }
    }
    part[wave][d] = x;
  }
  __syncthreads();
  // bk = b * kv_heads + kvh; head kvh * group + r % group of sequence b
  const int64_t at = (bk * group + r % group) * t_q + r / group;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int d = threadIdx.x;
  if (d < hd_v) T::store(out + at * hd_v, d, total == 0.f ? 0.f : ((part[0][d] + part[1][d]) + (part[2][d] + part[3][d])) * inv);
  if (threadIdx.x == 0) lse[at] = total == 0.f ? -__builtin_inff() : (base - up) * ATT_LN2 + logf(total);
}

template <typename T>
int join(const AttendArgs& a, const float* totals, const float* stats, int64_t splits, float up) {
  const int64_t rows_all = a.batch * a.heads * a.t_q;
  if (rows_all > 0x7fffffff || splits > JOIN_MOST) return fail(LIMN_HIP_EUNSUPPORTED, "attend: %lld rows exceed one launch", (long long)rows_all);
  hipLaunchKernelGGL((attend_join<T>), dim3((unsigned)rows_all), dim3(256), 0, a.stream, totals, stats, (typename T::Storage*)a.o0, (float*)a.o1,
                     rows_all, (int)splits, (int)a.group(), (int)a.t_q, (int)a.hd_v, up);
  return check_hip(hipGetLastError(), "joining attention's splits");
}

// dk and dv of the key rows: the parts' totals added in order and rounded (4 elements a thread), blocks with one that is
// not finite flagged.
template <typename T>
__global__ __launch_bounds__(256) void attend_join_keys(const float* __restrict__ partial, int parts, typename T::Storage* __restrict__ dk,
                                                        typename T::Storage* __restrict__ dv, int* __restrict__ odd, int64_t elements, int hd, int t_k) {
  const int64_t i = (blockIdx.x * (int64_t)256 + threadIdx.x) * 4;
  if (i >= elements) return;
  const float* at = partial + blockIdx.y * elements + i;
  f32x4 v = *(const f32x4*)at;
#pragma unroll 4
  for (int k = 1; k < parts; k++) v += *(const f32x4*)(at + 2 * k * elements);
  typename T::Storage* o = blockIdx.y ? dv : dk;
#pragma unroll
  for (int e = 0; e < 4; e++) T::store(o, i + e, v[e]);
  const f32x4 zero = v * 0.f;
  if (zero[0] + zero[1] + zero[2] + zero[3] != 0.f) {
    const int64_t row = i / hd, bk = row / t_k;
    atomicOr(odd + bk * ((t_k + ATT_ROWS - 1) / ATT_ROWS) + (row - bk * t_k) / ATT_ROWS, 1);
  }
}

template <typename T>
int join_keys(const AttendArgs& a, const FastArgs& kv) {
  const int64_t elements = a.batch * a.kv_heads * a.t_k * a.hd, groups = (elements / 4 + 255) / 256;
  hipLaunchKernelGGL((attend_join_keys<T>), dim3((unsigned)groups, 2), dim3(256), 0, a.stream, kv.partial, kv.head_parts * kv.tile_parts,
                     (typename T::Storage*)a.o1, (typename T::Storage*)a.o2, kv.odd, elements, (int)a.hd, (int)a.t_k);
  return check_hip(hipGetLastError(), "joining attention's key parts");
}

constexpr int64_t FILL = 512;  // workgroups that give every CU two

// Parts of the keys a general forward is cut into: rows in too few tiles to fill the GPU walk long
// sequences in parts of at least 8 key tiles (two a wave).
int64_t general_splits(const AttendArgs& a) {
  const int64_t blocks = a.batch * a.kv_heads * ((a.group() * a.t_q + 31) / 32), tiles = (a.t_k + 31) / 32;
  int64_t splits = (FILL + blocks - 1) / blocks;
  splits = splits < tiles / 8 ? splits : tiles / 8;
  return splits > 1 ? splits : 1;
}

int64_t split_bytes(const AttendArgs& a, int64_t splits) {
  const int64_t rows = a.batch * a.heads * a.t_q;
  return splits > 1 ? attend_align(splits * rows * a.hd_v * 4) + attend_align(splits * rows * 8) : 0;
}

int check_attend(const char* name, const AttendArgs& a) {
  if (a.dtype != LIMN_HIP_FLOAT32 && a.dtype != LIMN_HIP_FLOAT16 && a.dtype != LIMN_HIP_BFLOAT16)
    return fail(LIMN_HIP_EUNSUPPORTED, "%s: takes float32, float16 or bfloat16, not dtype code %d", name, a.dtype);
  if (a.batch < 1 || a.heads < 1 || a.kv_heads < 1 || a.t_q < 1 || a.t_k < 1 || a.hd < 1 || a.hd_v < 1)
    return fail(LIMN_HIP_EINVAL, "%s: sizes must be positive (batch %lld, heads %lld, kv_heads %lld, t_q %lld, t_k %lld, hd %lld, hd_v %lld)", name,
                (long long)a.batch, (long long)a.heads, (long long)a.kv_heads, (long long)a.t_q, (long long)a.t_k, (long long)a.hd, (long long)a.hd_v);
  if (a.heads % a.kv_heads != 0)
    return fail(LIMN_HIP_EINVAL, "%s: %lld query heads do not share %lld key heads evenly", name, (long long)a.heads, (long long)a.kv_heads);
  if (a.t_q > a.t_k && (a.causal || a.documents != nullptr || a.lengths != nullptr))
    return fail(LIMN_HIP_EINVAL, "%s: the queries are the last of the keys' positions: %lld queries and %lld keys", name, (long long)a.t_q, (long long)a.t_k);
  // the kernels' constants are floats: a scale or a cap past this, or a cap below its inverse, would be an infinity or a 0 there
  const double most = 0x1p120;
  if (!(fabs(a.scale) <= most)) return fail(LIMN_HIP_EINVAL, "%s: scale must be finite, between -2^120 and 2^120", name);
  if (a.softcap != 0 && !(a.softcap >= 1 / most && a.softcap <= most))
    return fail(LIMN_HIP_EINVAL, "%s: softcap must be positive, between 2^-120 and 2^120, or 0 for none", name);
  if (a.prefix != nullptr && !a.causal) return fail(LIMN_HIP_EINVAL, "%s: a prefix opens keys that causality hides; the call is not causal", name);
  if (a.hd > 256 || a.hd_v > 256) return fail(LIMN_HIP_EUNSUPPORTED, "%s: no kernel for head dims %lld and %lld (at most 256)", name, (long long)a.hd, (long long)a.hd_v);
  // positions and packed rows are 32-bit in the kernels; element offsets are 64-bit
  const int64_t size = (int64_t)1 << 30;
  if (a.t_k > size || a.t_q > size / a.group() || a.heads > size || a.batch > ((int64_t)1 << 40) / a.heads / (a.t_q > a.t_k ? a.t_q : a.t_k))
    return fail(LIMN_HIP_EUNSUPPORTED, "%s: sizes out of range", name);
  return LIMN_HIP_OK;
}

int check_pointers(const char* name, const AttendArgs& a, bool backward) {
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.o0 == nullptr || a.o1 == nullptr) return fail(LIMN_HIP_EINVAL, "%s: null buffer", name);
  if (backward && (a.out == nullptr || a.lse == nullptr || a.dout == nullptr || a.o2 == nullptr)) return fail(LIMN_HIP_EINVAL, "%s: null buffer", name);
  const uintptr_t size = a.dtype == LIMN_HIP_FLOAT32 ? 4 : 2;
  const uintptr_t typed = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.o0 | (uintptr_t)a.out | (uintptr_t)a.dout | (uintptr_t)a.o2 | (backward ? (uintptr_t)a.o1 : 0);
  const uintptr_t words = (uintptr_t)a.slopes | (uintptr_t)a.documents | (uintptr_t)a.prefix | (uintptr_t)a.lengths | (uintptr_t)a.lse | (backward ? 0 : (uintptr_t)a.o1);
  if (typed % size != 0 || words % 4 != 0) return fail(LIMN_HIP_EINVAL, "%s: buffers must be aligned to their element size", name);
  if (a.workspace_bytes < 0) return fail(LIMN_HIP_EINVAL, "%s: negative workspace size", name);
  return LIMN_HIP_OK;
}

// ---- the tiled kernels ----

int64_t granules_of(const AttendArgs& a) { return (a.t_k + 31) / 32; }
int64_t row_blocks(const AttendArgs& a) { return a.batch * a.heads * ((a.t_q + ATT_ROWS - 1) / ATT_ROWS); }
int64_t key_blocks(const AttendArgs& a) { return a.batch * a.kv_heads * ((a.t_k + ATT_ROWS - 1) / ATT_ROWS); }

// float32 calls go to the tiles of 128 rows where the general kernels, with a workgroup for every 32, have more than
// one for a CU; a backward, whose few key blocks are cut into parts, from half as many on. Causal, forward + backward, tiled
// against general at 64 dims: 8 heads x 256 rows 23 + 65 against 18 + 56 us, 8 x 512 37 + 88 against 27 + 98, 2 x 4096 223 +
// 413 against 134 + 655, 16 x 1024 65 + 154 against 107 + 356, 64 x 1024 94 + 256 against 424 + 1393; at 128 dims 8 x 256
// 38 + 107 against 29 + 104, 8 x 512 63 + 142 against 43 + 177, 16 x 1024 117 + 253 against 184 + 646.
bool f32_rows(const AttendArgs& a, bool backward) {
  const int64_t tiles = a.batch * a.heads * ((a.t_q + 31) / 32);
  return backward ? tiles >= 128 : tiles > 256;
}

// Sizes these kernels serve: 16-byte rows; the tiled ones also need a head's rows within 32-bit byte
// offsets and few enough streamed tiles for a block's list of them.
bool row_sizes(const AttendArgs& a) { return a.hd == a.hd_v && a.hd % (a.dtype == LIMN_HIP_FLOAT32 ? 4 : 8) == 0 && a.hd <= 128; }
bool half_sizes(const AttendArgs& a) { return a.dtype != LIMN_HIP_FLOAT32 && row_sizes(a); }
bool fast_sizes(const AttendArgs& a, bool backward) {
  return row_sizes(a) && a.t_q <= (1 << 17) && a.t_k <= (1 << 17) && (a.dtype != LIMN_HIP_FLOAT32 || f32_rows(a, backward));
}

bool aligned16(const AttendArgs& a, bool backward) {
  const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.o0 | (backward ? (uintptr_t)a.o1 | (uintptr_t)a.o2 | (uintptr_t)a.out | (uintptr_t)a.dout : 0);
  return at % 16 == 0;
}

// Forward calls that share their keys' bytes between the heads of a group and split long caches (attend_token.hip): of fewer
// queries than half a tiled block's 128 rows, and of a part of a sequence against a long cache in so few blocks that the
// tiled kernel would leave CUs idle. 32768 keys x 128, tiled against these: 128 queries of 8 heads 642 and 90 us, of 32
// over 8 key heads 646 and 186, 512 of 32 (128 blocks) 646 and 637; 1024 keys, 128 of 8: 30 and 31 (64 dims 26 and 20).
bool token_sizes(const AttendArgs& a) { return half_sizes(a) && (a.t_q < 64 || (row_blocks(a) < 128 && a.t_k >= 1024 && a.t_q <= a.t_k / 4)); }

// A call of such sizes goes to them where every buffer is 16-byte aligned and the scale positive: the forward's
// reference point is taken over unscaled scores, and moves when one passes it by 8 / (scale log2 e), which must be a number.
bool fast_call(const AttendArgs& a, bool backward) { return fast_sizes(a, backward) && a.scale >= 0x1p-100 && aligned16(a, backward); }

// Parts of the queries that a call with fewer key blocks than fill the GPU (two workgroups a CU up to 64 half-width
// dims, one else) cuts its dK/dV pass into, the heads of a group first: at least 4 tiles each. The backward of 16 heads
// over 2 key heads, 2048 x 128 bf16 causal, 505 -> 154 us; 12 over 3, 901 x 80 float32, 862 -> 235; 16 over 16,
// 512 x 64 bf16, whose parts are short, 41.0 -> 41.8.
struct KeyParts {
  int heads, tiles;
};
KeyParts key_parts(const AttendArgs& a) {
  const int64_t fill = a.dtype != LIMN_HIP_FLOAT32 && a.hd <= 64 ? 512 : 256, tiles = (a.t_q + 63) / 64;
  int64_t want = fill / key_blocks(a);
  if (want > a.group() * tiles / 4) want = a.group() * tiles / 4;
  if (want < 2) return {1, 1};
  const int64_t heads = want < a.group() ? want : a.group();
  return {(int)heads, (int)(want / heads)};
}
int64_t key_parts_bytes(const AttendArgs& a) {
  const KeyParts p = key_parts(a);
  return p.heads * p.tiles > 1 ? p.heads * p.tiles * 2 * a.batch * a.kv_heads * a.t_k * a.hd * 4 : 0;
}

// Bytes of dS between the backward's passes past 64 half-width dims, 0 for none: 2 a pair of positions, whether it is seen
// or not, up to HANDED_MOST, a hundredth of the memory; longer calls compute the scores a second time instead. Backward of
// 4 x 16 heads over 4 key heads x 4096 x 128, capped: 1163 us so, 1237 computed twice; 8 x 12 over 6 x 1021 x 80: 144
// and 149; 16 x 16 x 300 x 128: 96 and 101; 8 x 16 x 4096 x 128 with documents of 1024 (4 GiB, past the limit): 1081 and 1104.
constexpr int64_t HANDED_MOST = (int64_t)5 << 29;
int64_t key_tiles(const AttendArgs& a) { return (a.t_k + ATT_ROWS - 1) / ATT_ROWS * 2; }  // whole key blocks
int64_t handed_bytes(const AttendArgs& a) {
  if (!half_sizes(a) || a.hd <= 64 || row_blocks(a) > HANDED_MOST / (64 * ATT_ROWS * 2) / key_tiles(a)) return 0;
  return row_blocks(a) * key_tiles(a) * 64 * ATT_ROWS * 2;
}

// flags of the blocks, the documents' ranges, and for the backward delta
int64_t fast_workspace(const AttendArgs& a, bool backward) {
  if (!fast_sizes(a, backward)) return 0;
  int64_t need = attend_align(row_blocks(a) * 4) + attend_align(a.batch * granules_of(a) * 16);
  if (backward) need += attend_align(key_blocks(a) * 4) + attend_align(a.batch * a.heads * a.t_q * 4) + attend_align(key_parts_bytes(a)) + attend_align(handed_bytes(a));
  return need;
}

// Heads in a group of one XCD (att_head_and_block): 4, or 2 in a backward whose sequences differ in work by documents or
// lengths, so that each XCD has some of every sequence (8 x 16 heads x 4096 x 128, documents of 1024: backward 1124
// with 4 and 1096 with 2 us, forward 394 and 400); fewer heads than give each XCD two groups go alone, and fewer
// than 8, or a few that 8 does not divide, in turn.
int head_group(const AttendArgs& a, int64_t heads, bool backward) {
  int group = backward && (a.documents != nullptr || a.lengths != nullptr) ? 2 : 4;
  while (group > 1 && heads < 16 * group) group /= 2;
  return heads < 8 || (heads < 64 && heads % (8 * group) != 0) ? 0 : group;
}

#define LIMN_ATTEND_PASS(PASS, G)                                       \
  (a.dtype == LIMN_HIP_FLOAT32 ? launch_attend_##PASS##_parts(G, ra, a.stream) \
                               : (a.hd <= 64 ? launch_attend_##PASS##_64 : a.hd <= 96 ? launch_attend_##PASS##_96 : launch_attend_##PASS##_128)(G, ra, a.dtype, a.stream))

int launch_fast(const AttendArgs& a, bool backward) {
  const RuleArgs ra = rule_args(a);
  char* at = (char*)a.workspace;
  auto take = [&](int64_t bytes) {
    char* p = at;
    at += attend_align(bytes);
    return p;
  };
  int* odd = (int*)take(row_blocks(a) * 4);
  int4* ranges = (int4*)take(a.batch * granules_of(a) * 16);
  FastArgs g = {};
  g.q = (const u16*)a.q, g.k = (const u16*)a.k, g.v = (const u16*)a.v, g.out = (const u16*)a.out, g.dout = (const u16*)a.dout;
  g.lse_in = a.lse, g.o0 = (u16*)a.o0, g.odd = odd, g.ranges = a.documents != nullptr ? ranges : nullptr;
  g.batch = a.batch, g.heads = (int)a.heads, g.kv_heads = (int)a.kv_heads, g.hd = (int)a.hd, g.granules = (int)granules_of(a), g.scale = (float)a.scale;
  g.head_group = head_group(a, a.batch * a.heads, backward);
  int rc = LIMN_HIP_OK;
  if (a.documents != nullptr && (rc = launch_attend_ranges(ra, ranges, a.batch, g.granules, a.stream)) != LIMN_HIP_OK) return rc;
  // without causality and documents a hidden key is one past the live ones, which reads as zeros; but float32's parts do
  // not hold infinities, and float16's score gradients may overflow where the result does not
  const bool mend = a.causal || a.documents != nullptr || a.dtype == LIMN_HIP_FLOAT32 || (backward && a.dtype == LIMN_HIP_FLOAT16);
  if (!backward) {
    g.lse = (float*)a.o1;
    rc = LIMN_ATTEND_PASS(fwd, g);
    return rc != LIMN_HIP_OK || !mend ? rc : launch_attend_mend_fwd(g, ra, a.dtype, a.stream);
  }
  FastArgs kv = g;
  kv.odd = (int*)take(key_blocks(a) * 4);
  g.delta = kv.delta = (float*)take(a.batch * a.heads * a.t_q * 4);
  kv.o0 = (u16*)a.o1;
  kv.o1 = (u16*)a.o2;
  kv.head_group = head_group(a, a.batch * a.kv_heads, backward);
  const KeyParts parts = key_parts(a);
  kv.head_parts = parts.heads, kv.tile_parts = parts.tiles;
  kv.partial = parts.heads * parts.tiles > 1 ? (float*)take(key_parts_bytes(a)) : nullptr;
  g.row_blocks = kv.row_blocks = (int)((a.t_q + ATT_ROWS - 1) / ATT_ROWS);
  g.key_tiles = kv.key_tiles = (int)key_tiles(a);
  g.ds = kv.ds = handed_bytes(a) > 0 ? (u16*)take(handed_bytes(a)) : nullptr;
  rc = g.ds != nullptr ? launch_attend_delta(g, a.batch * a.heads * a.t_q, a.dtype, a.stream) : LIMN_ATTEND_PASS(dq, g);
  if (rc != LIMN_HIP_OK) return rc;
  rc = LIMN_ATTEND_PASS(dkv, kv);
  if (rc == LIMN_HIP_OK && g.ds != nullptr) rc = LIMN_ATTEND_PASS(dq, g);
  if (rc == LIMN_HIP_OK && kv.partial != nullptr)
    rc = a.dtype == LIMN_HIP_FLOAT32 ? join_keys<F32>(a, kv) : a.dtype == LIMN_HIP_FLOAT16 ? join_keys<F16>(a, kv) : join_keys<BF16>(a, kv);
  return rc != LIMN_HIP_OK || !mend ? rc : launch_attend_mend_bwd(g, kv, ra, a.dtype, a.stream);
}

// Enough for whichever kernels the call's buffers, rules and scale allow.
int64_t workspace_of(const AttendArgs& a, bool backward) {
  int64_t need = attend_general_workspace(a, backward);
  const int64_t fast = fast_workspace(a, backward), token = !backward && token_sizes(a) ? attend_token_workspace(a) : 0;
  if (fast > need) need = fast;
  return token > need ? token : need;
}

int launch(const AttendArgs& a, bool backward) {
  if (!backward && token_sizes(a) && a.documents == nullptr && aligned16(a, false)) return launch_attend_token(a);
  if (fast_call(a, backward) && (backward || a.t_q >= 64)) return launch_fast(a, backward);
  return backward ? launch_attend_general_bwd(a) : launch_attend_general_fwd(a);
}

int check_workspace(const char* name, const AttendArgs& a, bool backward) {
  const int64_t need = workspace_of(a, backward);
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need || (uintptr_t)a.workspace % 16 != 0))
    return fail(LIMN_HIP_EINVAL, "%s: needs a workspace of %lld bytes, 16-byte aligned", name, (long long)need);
  return LIMN_HIP_OK;
}

}  // namespace

int launch_attend_join(const AttendArgs& a, const float* totals, const float* stats, int64_t splits, float up) {
  if (a.dtype == LIMN_HIP_FLOAT32) return join<F32>(a, totals, stats, splits, up);
  return a.dtype == LIMN_HIP_FLOAT16 ? join<F16>(a, totals, stats, splits, up) : join<BF16>(a, totals, stats, splits, up);
}

int64_t attend_general_workspace(const AttendArgs& a, bool backward) {
  return backward ? attend_align(a.batch * a.heads * a.t_q * 4) : split_bytes(a, general_splits(a));
}

int launch_attend_general_fwd(const AttendArgs& a) {
  const int64_t splits = general_splits(a);
  if (a.dtype == LIMN_HIP_FLOAT32) return attend_general_fwd_f32(a, splits);
  return a.dtype == LIMN_HIP_FLOAT16 ? attend_general_fwd_f16(a, splits) : attend_general_fwd_bf16(a, splits);
}

int launch_attend_general_bwd(const AttendArgs& a) {
  if (a.dtype == LIMN_HIP_FLOAT32) return attend_general_bwd_f32(a);
  return a.dtype == LIMN_HIP_FLOAT16 ? attend_general_bwd_f16(a) : attend_general_bwd_bf16(a);
}

}  // namespace limn

using namespace limn;

extern "C" {

int64_t limn_hip_attend_workspace(int dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t t_q, int64_t t_k, int64_t hd,
                                  int64_t hd_v, int backward) {
  AttendArgs a = {};
  a.dtype = dtype, a.batch = batch, a.heads = heads, a.kv_heads = kv_heads, a.t_q = t_q, a.t_k = t_k, a.hd = hd, a.hd_v = hd_v;
  if (check_attend("attend_workspace", a) != LIMN_HIP_OK) return 0;
  return workspace_of(a, backward != 0);
}

int limn_hip_attend_fwd(const void* q, const void* k, const void* v, const void* slopes, const void* documents, const void* prefix,
                        const void* lengths, void* out, void* lse, int dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t t_q,
                        int64_t t_k, int64_t hd, int64_t hd_v, int causal, double scale, double softcap, void* workspace,
                        int64_t workspace_bytes, void* stream) {
  AttendArgs a = {q, k, v, (const float*)slopes, (const int*)documents, (const int*)prefix, (const int*)lengths, nullptr, nullptr, nullptr,
                  out, lse, nullptr, dtype, batch, heads, kv_heads, t_q, t_k, hd, hd_v, causal != 0, scale, softcap, workspace, workspace_bytes,
                  (hipStream_t)stream};
  int rc = check_attend("attend_fwd", a);
  if (rc == LIMN_HIP_OK) rc = check_pointers("attend_fwd", a, false);
  if (rc == LIMN_HIP_OK) rc = check_workspace("attend_fwd", a, false);
  return rc != LIMN_HIP_OK ? rc : launch(a, false);
}

int limn_hip_attend_bwd(const void* q, const void* k, const void* v, const void* slopes, const void* documents, const void* prefix,
                        const void* lengths, const void* out, const void* lse, const void* dout, void* dq, void* dk, void* dv, int dtype,
                        int64_t batch, int64_t heads, int64_t kv_heads, int64_t t_q, int64_t t_k, int64_t hd, int64_t hd_v, int causal,
                        double scale, double softcap, void* workspace, int64_t workspace_bytes, void* stream) {
  AttendArgs a = {q, k, v, (const float*)slopes, (const int*)documents, (const int*)prefix, (const int*)lengths, out, (const float*)lse, dout,
                  dq, dk, dv, dtype, batch, heads, kv_heads, t_q, t_k, hd, hd_v, causal != 0, scale, softcap, workspace, workspace_bytes,
                  (hipStream_t)stream};
  int rc = check_attend("attend_bwd", a);
  if (rc == LIMN_HIP_OK) rc = check_pointers("attend_bwd", a, true);
  if (rc == LIMN_HIP_OK) rc = check_workspace("attend_bwd", a, true);
  return rc != LIMN_HIP_OK ? rc : launch(a, true);
}

}  // extern "C"
