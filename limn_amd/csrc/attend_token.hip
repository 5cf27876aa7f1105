// Attention with score rules for few queries against a cache (the single-token form, and parts of a sequence against
// what came before): half widths, hd == hd_v up to 128 in multiples of 8, no documents.
//
// What bounds it is reading k and v once (2 hd bytes each a key): everything is laid out for that.
//  - The queries of every head that shares a key head are rows of one tile (16 NR packed rows), so k and v are
//    read once for all of them.
//  - A wave takes 32 keys at a time and reads them from memory straight into the operands of
//    v_mfma_f32_16x16x32, no LDS and no barrier in the loop. K: lane (n = lane % 16, g = lane / 16) reads
//    dims 32 s + 8 g .. + 7 of key n: 64 consecutive bytes a key. V: the lane reads dims W n .. W n + W - 1
//    (W = D / 16) of keys 4 g + j and 16 + 4 g + j, whole rows of 16 lanes; S^T = K Q^T leaves exactly those
//    keys' weights in the lane, so they are the second product's B operand as they stand, and its A operand
//    for dims W m + e is element e of the lane's 8 keys (a byte permute each).
//  - The next 32 keys' loads are issued as soon as the registers they go to are free: K behind the scores, V
//    behind the second product. 16 KB a wave are in flight at D = 128, and 8 or more waves a CU.
//  - A key that some queries of a tile see and others do not (the last t_q ones, a prefix) may hold an infinity or
//    a NaN, which a weight of 0 does not hide: a call of more than one query is followed by a kernel that
//    computes rows with results that are not finite again in float (launch_attend_mend_rows).
//  - 32 sequences of up to 8192 positions, 32 heads over 8 key heads x 128 (672 MB): 141 us, 4.8 TB/s, what a copy
//    reaches; one of 1000 positions, 8 heads x 64: 9.3 us, one launch's latency and the call.
//  - Long caches are cut into parts over workgroups, joined by a second kernel (attend_join) in order; short
//    ones go to workgroups of 16 waves, joined in LDS, where one launch is faster than two.

#include "attend_fast.h"

namespace limn {
namespace {

constexpr int TOK_KEYS = 32;  // keys a wave takes at a time

template <typename T>
__device__ __forceinline__ f32x4 mfma16(u16x8 a, u16x8 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma16<BF16>(u16x8 a, u16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma16<F16>(u16x8 a, u16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

struct TokenArgs {
  const u16* q;
  const u16* k;
  const u16* v;
  u16* out;
  float* lse;
  float* totals;  // parts > 1: (parts, batch * kv_heads * rows, hd)
  float* stats;   // (parts, batch * kv_heads * rows, 2)
  int64_t batch;
  int heads, kv_heads, hd, rows, row_tiles, parts, part_tiles;  // rows = group * t_q; tiles of 32 keys in a part
};

// the 4 lanes groups of a column combined
__device__ __forceinline__ float col_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float col_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <int W>
struct VChunk;  // W consecutive 16-bit elements
template <>
struct VChunk<8> {
  u16x8 x;
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int off) { x = __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0)); }
};
template <>
struct VChunk<4> {
  u16x4 x;
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int off) { x = __builtin_bit_cast(u16x4, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0)); }
};

template <typename T, int D, int NR, int waves>
__global__ __launch_bounds__(64 * waves, waves == 4 ? 2 : 1) void attend_token(TokenArgs a, RuleArgs ra) {
  constexpr int W = D / 16, KS = D / 32;
  __shared__ float lds[waves * 16 * 17 + waves * NR * 32];
  constexpr float UP = std::is_same<T, F16>::value ? 7.f : 0.f;  // float16 weights times 2^7: see shift_of in attend_mfma.h
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  // parts of one key head apart by the number of key heads: neighbours in launch order read different heads
  int64_t id = blockIdx.x;
  const int64_t bk = id % (a.batch * a.kv_heads);
  id /= a.batch * a.kv_heads;
  const int part = (int)(id % a.parts), rt = (int)(id / a.parts);
  const int64_t b = bk / a.kv_heads;
  const int kvh = (int)(bk - b * a.kv_heads), group = a.heads / a.kv_heads;
  const Rules r = rules_of(ra, b);
  const u16* kbase = a.k + bk * (int64_t)r.t_k * a.hd;
  const u16* vbase = a.v + bk * (int64_t)r.t_k * a.hd;

  // this lane's rows: packed row -> query, head
  int p[NR];
  float slope2[NR];
  int64_t at[NR];
  bool there[NR];
  u16x8 qf[NR][KS];
  f32x4 acc[NR][W];
  float m[NR], l[NR];
  int pmin = 0x7fffffff, pmax = -0x7fffffff;
#pragma unroll
  for (int t = 0; t < NR; t++) {
    const int row = rt * 16 * NR + t * 16 + n;
    there[t] = row < a.rows;
    const int i = there[t] ? row / group : 0, head = kvh * group + (there[t] ? row % group : 0);
    p[t] = r.off + i;
    if (there[t]) {
      pmin = min(pmin, p[t]);
      pmax = max(pmax, p[t]);
    }
    at[t] = (b * a.heads + head) * (int64_t)r.t_q + i;
    slope2[t] = ra.slopes != nullptr ? ra.slopes[head] * ATT_LOG2E : 0.f;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const int d = 32 * s + 8 * g;
      qf[t][s] = there[t] && d < a.hd ? *(const u16x8*)(a.q + at[t] * a.hd + d) : u16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
#pragma unroll
    for (int e = 0; e < W; e++) acc[t][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[t] = -__builtin_inff();
    l[t] = 0.f;
  }
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) {
    pmin = min(pmin, __shfl_xor(pmin, x));
    pmax = max(pmax, __shfl_xor(pmax, x));
  }
  pmin = __builtin_amdgcn_readfirstlane(pmin);
  pmax = __builtin_amdgcn_readfirstlane(pmax);

  int kend = r.len;
  if (r.causal) kend = min(kend, max(pmax + 1, r.pre));
  const int tiles = kend > 0 ? (kend + TOK_KEYS - 1) / TOK_KEYS : 0;
  const int first = part * a.part_tiles, last = min(tiles, first + a.part_tiles);

  u16x8 kr[2][KS];
  VChunk<W> vr[8];
  // a tile's bytes from its own base, so that a cache of any length is reached by 32-bit offsets; keys past
  // the live ones read as zeros
  auto rsrc = [&](const u16* base, int k0) __attribute__((always_inline)) {
    const int left = r.len - k0;
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)k0 * a.hd), (short)0, (left < TOK_KEYS ? left : TOK_KEYS) * a.hd * 2, 0x00020000);
  };
  auto load_k = [&](int kt) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t res = rsrc(kbase, kt * TOK_KEYS);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const int d = 32 * s + 8 * g;
        kr[t][s] = __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(res, d < a.hd ? ((16 * t + n) * a.hd + d) * 2 : 0x7ffffff0, 0, 0));
      }
  };
  auto load_v = [&](int kt) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t res = rsrc(vbase, kt * TOK_KEYS);
#pragma unroll
    for (int j = 0; j < 8; j++) vr[j].load(res, W * n < a.hd ? ((16 * (j >> 2) + 4 * g + (j & 3)) * a.hd + W * n) * 2 : 0x7ffffff0);
  };
  int kt = first + wave;
  if (kt < last) {
    load_k(kt);
    load_v(kt);
  }
  for (; kt < last; kt += waves) {
    const int k0 = kt * TOK_KEYS;
    const bool more = kt + waves < last;
    f32x4 s[NR][2];
#pragma unroll
    for (int t = 0; t < NR; t++)
#pragma unroll
      for (int c = 0; c < 2; c++) s[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int t = 0; t < NR; t++) s[t][c] = mfma16<T>(kr[c][ks], qf[t][ks], s[t][c]);
    if (more) load_k(kt + waves);
    const bool edge = k0 + TOK_KEYS > r.len || (r.causal && k0 + TOK_KEYS - 1 > pmin && k0 + TOK_KEYS - 1 >= r.pre);
    u16x8 pb[NR];
#pragma unroll
    for (int t = 0; t < NR; t++) {
      float y[8], mx = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = s[t][j >> 2][j & 3];
      if (r.cap_out > 0.f) {
        cap_scores<8>(y, r);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] *= r.c2;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int key = k0 + 16 * (j >> 2) + 4 * g + (j & 3);
        float x = fmaf(-slope2[t], fabsf((float)(p[t] - key)), y[j]);
        if (edge) x = sees(r, p[t], key) ? x : -__builtin_inff();
        y[j] = x;
        mx = fmaxf(mx, x);
      }
      if (__any(mx > m[t] + 8.f)) {
        mx = col_max(mx);
        const float up = fmaxf(m[t], mx), alpha = up == -__builtin_inff() ? 1.f : fast_exp2(m[t] - up);
        l[t] *= alpha;
#pragma unroll
        for (int e = 0; e < W; e++) acc[t][e] *= alpha;
        m[t] = up;
      }
      const float base = (m[t] == -__builtin_inff() ? 0.f : m[t]) - UP;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        y[j] = fast_exp2(y[j] - base);
        l[t] += y[j];
      }
      const u32x4 w = {T::pack2(y[0], y[1]), T::pack2(y[2], y[3]), T::pack2(y[4], y[5]), T::pack2(y[6], y[7])};
      pb[t] = __builtin_bit_cast(u16x8, w);
    }
#pragma unroll
    for (int e = 0; e < W; e++) {
      u16x8 va;
#pragma unroll
      for (int j = 0; j < 8; j++) va[j] = vr[j].x[e];
#pragma unroll
      for (int t = 0; t < NR; t++) acc[t][e] = mfma16<T>(va, pb[t], acc[t][e]);
    }
    if (more) load_v(kt + waves);
  }

  // join the waves in order, one 16-dim slice of one row tile at a time
  float* sm = lds + waves * 16 * 17;
#pragma unroll
  for (int t = 0; t < NR; t++) {
    l[t] = col_sum(l[t]);
    if (g == 0) {
      sm[(wave * NR + t) * 32 + n] = m[t];
      sm[(wave * NR + t) * 32 + 16 + n] = l[t];
    }
  }
  __syncthreads();
  const int64_t rows_all = a.batch * a.kv_heads * (int64_t)a.rows;
#pragma unroll
  for (int t = 0; t < NR; t++) {
    float top = -__builtin_inff(), total = 0.f;
    for (int w = 0; w < waves; w++) top = fmaxf(top, sm[(w * NR + t) * 32 + n]);
    for (int w = 0; w < waves; w++) {
      const float mw = sm[(w * NR + t) * 32 + n], lw = sm[(w * NR + t) * 32 + 16 + n];
      total += mw == -__builtin_inff() ? lw : lw * fast_exp2(mw - top);
    }
    const float factor = m[t] == -__builtin_inff() ? 1.f : fast_exp2(m[t] - top);
    const int row = rt * 16 * NR + t * 16 + n;
    if (wave == 0 && g == 0 && there[t]) {
      if (a.parts > 1) {
        float* st = a.stats + (part * rows_all + bk * a.rows + row) * 2;
        st[0] = top;
        st[1] = total;
      } else {
        a.lse[at[t]] = total == 0.f ? -__builtin_inff() : ((top == -__builtin_inff() ? 0.f : top) - UP) * ATT_LN2 + logf(total);
      }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int e = 0; e < W; e++) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; i++) lds[(wave * 16 + 4 * g + i) * 17 + n] = acc[t][e][i] * factor;  // dim W (4 g + i) + e
      __syncthreads();
      if (wave < 4) {  // 16 dims x 16 rows: wave w takes dims 4 w + g of row n
        const int dd = 4 * wave + g, d = W * dd + e;
        float x = 0.f;
        for (int w = 0; w < waves; w++) x += lds[(w * 16 + dd) * 17 + n];
        if (there[t] && d < a.hd) {
          if (a.parts > 1)
            a.totals[(part * rows_all + bk * a.rows + row) * a.hd + d] = x;
          else
            T::store(a.out + at[t] * a.hd, d, total == 0.f ? 0.f : x * inv);
        }
      }
    }
    __syncthreads();
  }
}

// Waves of a workgroup that has a row tile to itself: as many as its registers allow without spills.
template <int D, int NR>
constexpr int LONE_WAVES = D == 64 && NR == 1 ? 16 : 8;

struct TokenPlan {
  int nr, waves, parts, part_tiles, row_tiles;
};

// Row tiles of 16 where one holds all packed rows or the last half of a second would be idle, else of 32. Up to
// 64 key tiles go to one workgroup of 16 waves a row tile while such workgroups leave waves free; longer
// caches to workgroups of 4 waves, in as many parts as give every CU four of them, each at least 8 key tiles.
TokenPlan token_plan(const AttendArgs& a) {
  TokenPlan p;
  const int64_t rows = a.group() * a.t_q, tiles = (a.t_k + TOK_KEYS - 1) / TOK_KEYS;
  p.nr = rows <= 16 ? 1 : 2;
  p.row_tiles = (int)((rows + 16 * p.nr - 1) / (16 * p.nr));
  const int64_t units = a.batch * a.kv_heads * p.row_tiles;
  p.waves = tiles <= 64 && units <= 256 ? 16 : 4;
  int64_t parts = p.waves == 16 ? 1 : 1024 / units;
  if (parts > tiles / 8) parts = tiles / 8;
  if (parts < 1) parts = 1;
  p.part_tiles = (int)((tiles + parts - 1) / parts);
  p.parts = (int)((tiles + p.part_tiles - 1) / p.part_tiles);
  return p;
}

template <typename T, int D, int NR>
int launch_token(const TokenArgs& t, const RuleArgs& ra, const TokenPlan& p, hipStream_t stream) {
  const int64_t blocks = t.batch * t.kv_heads * p.parts * p.row_tiles;
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "attend: %lld workgroups exceed one launch", (long long)blocks);
  if (p.waves == 4)
    hipLaunchKernelGGL((attend_token<T, D, NR, 4>), dim3((unsigned)blocks), dim3(256), 0, stream, t, ra);
  else
    hipLaunchKernelGGL((attend_token<T, D, NR, LONE_WAVES<D, NR>>), dim3((unsigned)blocks), dim3(64 * LONE_WAVES<D, NR>), 0, stream, t, ra);
  return check_hip(hipGetLastError(), "launching attention against a cache");
}

template <typename T>
int launch_token_type(const TokenArgs& t, const RuleArgs& ra, const TokenPlan& p, hipStream_t stream) {
  if (t.hd <= 64) return p.nr == 1 ? launch_token<T, 64, 1>(t, ra, p, stream) : launch_token<T, 64, 2>(t, ra, p, stream);
  return p.nr == 1 ? launch_token<T, 128, 1>(t, ra, p, stream) : launch_token<T, 128, 2>(t, ra, p, stream);
}

}  // namespace

int64_t attend_token_workspace(const AttendArgs& a) {
  const TokenPlan p = token_plan(a);
  const int64_t rows = a.batch * a.heads * a.t_q;
  return p.parts > 1 ? attend_align(p.parts * rows * a.hd * 4) + attend_align(p.parts * rows * 8) : 0;
}

int launch_attend_token(const AttendArgs& a) {
  const TokenPlan p = token_plan(a);
  const int64_t rows_all = a.batch * a.heads * a.t_q;
  float* totals = p.parts > 1 ? (float*)a.workspace : nullptr;
  float* stats = p.parts > 1 ? (float*)((char*)a.workspace + attend_align(p.parts * rows_all * a.hd * 4)) : nullptr;
  const TokenArgs t = {(const u16*)a.q, (const u16*)a.k, (const u16*)a.v, (u16*)a.o0, (float*)a.o1, totals, stats, a.batch, (int)a.heads, (int)a.kv_heads,
                       (int)a.hd, (int)(a.group() * a.t_q), p.row_tiles, p.parts, p.part_tiles};
  int rc = a.dtype == LIMN_HIP_BFLOAT16 ? launch_token_type<BF16>(t, rule_args(a), p, a.stream) : launch_token_type<F16>(t, rule_args(a), p, a.stream);
  if (rc == LIMN_HIP_OK && p.parts > 1) rc = launch_attend_join(a, totals, stats, p.parts, a.dtype == LIMN_HIP_FLOAT16 ? 7.f : 0.f);
  return rc == LIMN_HIP_OK && a.causal && a.t_q > 1 ? launch_attend_mend_rows(a) : rc;
}

}  // namespace limn
