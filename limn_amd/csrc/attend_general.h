// Attention with score rules in float arithmetic, for every storage type, head dim and alignment: the
// kernels that are right for every case, and the blocks the half-width kernels hand over to when a tile
// that is only partly visible holds an infinity or a NaN.
//
// A workgroup of 4 waves owns 32 resident rows (packed query rows, or keys for the dK/dV pass); the other
// side streams past in tiles of 32 that the waves take in turn, each wave with its own running totals,
// joined through LDS at the end in wave order. Every product is v_mfma_f32_32x32x2f32 with the resident
// rows on the N side, so a lane (n = lane % 32, h = lane / 32) owns resident row n:
//   S^T = K Q^T (forward, dQ pass) or S = Q K^T (dK/dV pass): both operands are read straight from memory,
//     4 consecutive dims a lane (dims 8 c + 4 h + e at step (c, e): the order of the contraction is free);
//   accumulator item i then holds streamed row 8 (i / 4) + 4 h + i % 4, which is exactly the pair of
//     rows (h = 0, 1) that step i of the next product contracts: its B operand is item i as it stands,
//     and its A operand one element X[streamed row][32 dt + n] a lane, 128 consecutive bytes a half-wave.
// Nothing is staged, so there is no barrier in the loop, and 64 workgroups already spread 8 heads x 256 rows over the GPU
// (float32 x 64, every rule: forward 22 us, backward 27 + 37, chains of loads and products). Where there are many, what
// bounds it is the reads: a wave's streamed tile serves 32 resident rows alone (64 heads x 2048 x 64 causal: forward 1248
// us, 27 of the 157 TFLOP/s that float32 products reach).
//
// A hidden pair contributes nothing, whatever stands in the hidden row: its probability is selected to 0,
// and where the streamed row of a product holds an infinity or a NaN (0 times which is NaN), the row's
// non-finite elements are taken out of the product and added only to the rows that see them (see add).
#pragma once

#include "attend_rules.h"

namespace limn {
namespace {

constexpr int GEN_THREADS = 256, GEN_WAVES = 4;
constexpr int GEN_LDS = GEN_WAVES * 32 * 33 + GEN_WAVES * 64;  // floats a block needs

__device__ __forceinline__ f32x16 gen_zero() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; i++) z[i] = 0.f;
  return z;
}

__device__ __forceinline__ f32x16 gen_mfma(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

// x combined with the same register of lane ^ 32
__device__ __forceinline__ float gen_pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float gen_pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The rows of a block: packed row r is query r / group of head head0 + r % group.
struct RowMap {
  int group, head0, rows;  // rows = group * t_q
  __device__ __forceinline__ int query(int r) const { return group == 1 ? r : r / group; }
  __device__ __forceinline__ int head(int r) const { return group == 1 ? head0 : head0 + r % group; }
  // element offset of row r in a (heads, t_q, width) matrix
  __device__ __forceinline__ int64_t at(int r, int t_q, int width) const { return ((int64_t)head(r) * t_q + query(r)) * width; }
};

// 4 consecutive elements of a row of `width`, zeros past its end or where the row is not there; `vec`: the
// width is a multiple of 4 and rows start on 4-element boundaries.
template <typename T>
__device__ __forceinline__ f32x4 gen_load4(const typename T::Storage* row, bool there, int d, int width, bool vec) {
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (!there) return x;
  if (vec) {
    if (d >= width) return x;
    if constexpr (sizeof(typename T::Storage) == 4) {
      x = *(const f32x4*)(row + d);
    } else {
      const u16x4 w = *(const u16x4*)(row + d);
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = T::unpack(w[e]);
    }
    return x;
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (d + e < width) x[e] = (float)T::load(row, d + e);
  return x;
}

template <typename T>
__device__ __forceinline__ float gen_load1(const typename T::Storage* row, bool there, int d, int width) {
  return there && d < width ? (float)T::load(row, d) : 0.f;
}

__device__ __forceinline__ bool gen_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// The score (log2 units) of a product, and the factor its cap takes off the gradient.
__device__ __forceinline__ float gen_score(const Rules& r, float x, float slope2, float far, float& bent) {
  float y = x * r.c2;
  bent = 1.f;
  if (r.cap_out > 0.f) {
    const float z = y * r.cap_un, t = tanhf(z);
    if (fabsf(z) > 0x1p-13f) y = t * r.cap_out;  // below, the score itself: z may be under float's normal numbers
    bent = fmaf(-t, t, 1.f);
  }
  return y - slope2 * far;
}

// acc += A^T B over the 32 streamed rows whose elements (at this lane's dim) are a[i], with the resident
// rows' factors p[i]; `vis` bit i: resident row n sees streamed row i (p[i] is 0 where it does not).
// `partly`: some pair of the tile is hidden. A non-finite element times a hidden row's 0 would be NaN, so
// in such tiles the finite elements are multiplied first, and what the others add (p a of the visible
// pairs alone: NaN, or infinities by the signs of a and p) is found from products of their indicators.
__device__ __forceinline__ void gen_add(f32x16& acc, const float (&a)[16], const float (&p)[16], unsigned vis, bool partly) {
  bool odd = false;
  if (partly) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 16; i++) bad |= !gen_finite(a[i]);
    odd = __any(bad);
  }
  if (!odd) {
#pragma unroll
    for (int i = 0; i < 16; i++) acc = gen_mfma(a[i], p[i], acc);
    return;
  }
  f32x16 sum = gen_zero(), all = gen_zero(), nan = gen_zero();
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const bool see = (vis >> i) & 1u;
    const float up = a[i] > 3.402823466e38f ? 1.f : a[i] < -3.402823466e38f ? -1.f : 0.f;
    const float way = see ? (p[i] > 0.f ? 1.f : p[i] < 0.f ? -1.f : 0.f) : 0.f;
    acc = gen_mfma(gen_finite(a[i]) ? a[i] : 0.f, p[i], acc);
    sum = gen_mfma(up, way, sum);
    all = gen_mfma(fabsf(up), fabsf(way), all);
    nan = gen_mfma(a[i] != a[i] ? 1.f : 0.f, see ? 1.f : 0.f, nan);
    nan = gen_mfma(fabsf(up), see && way == 0.f ? 1.f : 0.f, nan);
  }
#pragma unroll
  for (int e = 0; e < 16; e++) {
    if (all[e] > 0.f) acc[e] += fabsf(sum[e]) < all[e] ? __builtin_nanf("") : sum[e] > 0.f ? __builtin_inff() : -__builtin_inff();
    if (nan[e] > 0.f) acc[e] = __builtin_nanf("");
  }
}

// The 4 waves' accumulators of one 32-dim tile (lane n = row, items = dims), each times its row's factor,
// added in wave order; thread (row, quad of dims) gets 4 sums. `lds`: GEN_WAVES * 32 * 33 floats.
__device__ __forceinline__ f32x4 gen_join(const f32x16& acc, float factor, float* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 31, h = lane >> 5;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; i++) lds[(wave * 32 + n) * 33 + 8 * (i >> 2) + 4 * h + (i & 3)] = acc[i] * factor;
  __syncthreads();
  const int row = threadIdx.x >> 3, d = (threadIdx.x & 7) * 4;
  f32x4 x;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    x[e] = lds[row * 33 + d + e];
#pragma unroll
    for (int w = 1; w < GEN_WAVES; w++) x[e] += lds[(w * 32 + row) * 33 + d + e];
  }
  return x;
}

// The documents of a 32-key tile: lane n holds key k0 + n's (-1 past the live keys), and whether any of
// them can meet the rows' documents [lo, hi].
__device__ __forceinline__ int gen_key_doc(const Rules& r, int key) { return r.docs != nullptr && key < r.len ? r.docs[key] : (r.docs ? -1 : 0); }

// What a row tile knows of itself: each lane its row's position, document and slope, and the wave their ranges.
struct RowTile {
  int p, doc;
  float slope2;
  int pmin, pmax, dlo, dhi;
};

__device__ __forceinline__ int gen_min(int x) {
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) x = min(x, __shfl_xor(x, m));
  return x;
}
__device__ __forceinline__ int gen_max(int x) {
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) x = max(x, __shfl_xor(x, m));
  return x;
}

// (both halves of a wave hold the same rows, so ranges need the 32 lanes of one only)
__device__ __forceinline__ RowTile gen_row_tile(const Rules& r, const RuleArgs& ra, const RowMap& map, int row) {
  RowTile t;
  const bool there = row < map.rows;
  t.p = there ? r.off + map.query(row) : -1;
  t.doc = there ? query_doc(r, t.p) : -1;
  t.slope2 = there && ra.slopes ? ra.slopes[map.head(row)] * ATT_LOG2E : 0.f;
  t.pmin = __builtin_amdgcn_readfirstlane(gen_min(there ? t.p : 0x7fffffff));
  t.pmax = __builtin_amdgcn_readfirstlane(gen_max(there ? t.p : -0x7fffffff));
  t.dlo = __builtin_amdgcn_readfirstlane(gen_min(t.doc >= 0 ? t.doc : 0x7fffffff));
  t.dhi = __builtin_amdgcn_readfirstlane(gen_max(t.doc));
  return t;
}

// Whether no pair of a row tile and a key tile is visible, and whether every one is. kd: lane n's key
// document.
__device__ __forceinline__ bool gen_none(const Rules& r, const RowTile& t, int k0, int kd) {
  if (k0 >= r.len) return true;
  if (r.causal && k0 > t.pmax && k0 >= r.pre) return true;
  return r.docs != nullptr && !__any(kd >= 0 && kd >= t.dlo && kd <= t.dhi);
}
__device__ __forceinline__ bool gen_whole(const Rules& r, const RowTile& t, bool rows_there, int k0, int kd) {
  if (!rows_there || k0 + 32 > r.len) return false;
  if (r.causal && k0 + 31 > t.pmin && k0 + 31 >= r.pre) return false;
  return r.docs == nullptr || (__all(t.doc == t.dlo) && __all(kd == t.dlo));
}

// ---- forward --------------------------------------------------------------------------------------------

struct GenFwd {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;
  float* totals;  // split: (splits, batch * kv_heads * rows, hd_v), else nullptr
  float* stats;   // (splits, batch * kv_heads * rows, 2)
  int64_t batch;
  int heads, kv_heads, hd, hd_v, vec, splits;
};

// Packed rows [row0, row0 + 32) of key head kvh of sequence b, over part `split` of the key tiles.
template <typename T, int DT>
__device__ __forceinline__ void gen_fwd_block(const GenFwd& g, const RuleArgs& ra, const RowMap& map, int64_t b, int kvh, int row0,
                                              int split, float* lds) {
  typedef typename T::Storage S;
  constexpr int CH = DT * 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const Rules r = rules_of(ra, b);
  const int row = row0 + n;
  const bool there = row < map.rows;
  const RowTile t = gen_row_tile(r, ra, map, row);
  const S* q = (const S*)g.q + b * g.heads * (int64_t)r.t_q * g.hd;
  const S* k = (const S*)g.k + (b * g.kv_heads + kvh) * (int64_t)r.t_k * g.hd;
  const S* v = (const S*)g.v + (b * g.kv_heads + kvh) * (int64_t)r.t_k * g.hd_v;

  f32x4 qf[CH];
  f32x16 acc[DT];
#pragma unroll
  for (int c = 0; c < CH; c++) qf[c] = gen_load4<T>(q + (there ? map.at(row, r.t_q, g.hd) : 0), there, 8 * c + 4 * h, g.hd, g.vec);
#pragma unroll
  for (int dt = 0; dt < DT; dt++) acc[dt] = gen_zero();
  float m = -__builtin_inff(), l = 0.f;

  int kend = r.len;
  if (r.causal) kend = min(kend, max(t.pmax + 1, r.pre));
  const int tiles = kend > 0 ? (kend + 31) / 32 : 0;
  const int per = (tiles + g.splits - 1) / g.splits, last = min(tiles, (split + 1) * per);
  for (int kt = split * per + wave; kt < last; kt += GEN_WAVES) {
    const int k0 = kt * 32;
    const int kd = gen_key_doc(r, k0 + n);
    if (gen_none(r, t, k0, kd)) continue;
    const bool whole = gen_whole(r, t, row0 + 32 <= map.rows, k0, kd);
    const bool key_there = k0 + n < r.len;
    f32x16 s = gen_zero();
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const f32x4 a = gen_load4<T>(k + (int64_t)(k0 + n) * g.hd, key_there, 8 * c + 4 * h, g.hd, g.vec);
#pragma unroll
      for (int e = 0; e < 4; e++) s = gen_mfma(a[e], qf[c][e], s);
    }
    unsigned vis = 0xffffu;
    float p[16], mx = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int at = 8 * (i >> 2) + 4 * h + (i & 3), key = k0 + at;
      float bent;
      p[i] = gen_score(r, s[i], t.slope2, fabsf((float)(t.p - key)), bent);
      if (!whole) {
        const int d = __shfl(kd, at);
        const bool see = there & sees(r, t.p, key) & (t.doc >= 0) & (d == t.doc);
        p[i] = see ? p[i] : -__builtin_inff();
        if (!see) vis &= ~(1u << i);
      }
      mx = fmaxf(mx, p[i]);
    }
    mx = gen_pair_max(mx);
    // the reference point moves only when a score passes it by 8 (a factor of 256, which the float
    // totals carry as exactly), so that totals are rescaled rarely
    if (__any(mx > m + 8.f)) {
      const float up = fmaxf(m, mx), alpha = up == -__builtin_inff() ? 1.f : fast_exp2(m - up);
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; dt++) acc[dt] *= alpha;
      m = up;
    }
    const float base = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      p[i] = fast_exp2(p[i] - base);
      l += p[i];
    }
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
      float a[16];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int key = k0 + 8 * (i >> 2) + 4 * h + (i & 3);
        a[i] = gen_load1<T>(v + (int64_t)key * g.hd_v, key < r.len, 32 * dt + n, g.hd_v);
      }
      gen_add(acc[dt], a, p, vis, !whole);
    }
  }

  // join the waves: the largest reference point, the sums and totals brought to it
  float* sm = lds + GEN_WAVES * 32 * 33;
  l = gen_pair_sum(l);
  __syncthreads();
  if (h == 0) {
    sm[wave * 64 + n] = m;
    sm[wave * 64 + 32 + n] = l;
  }
  __syncthreads();
  float top = -__builtin_inff(), total = 0.f;
#pragma unroll
  for (int w = 0; w < GEN_WAVES; w++) top = fmaxf(top, sm[w * 64 + n]);
#pragma unroll
  for (int w = 0; w < GEN_WAVES; w++) {
    const float mw = sm[w * 64 + n], lw = sm[w * 64 + 32 + n];
    total += mw == -__builtin_inff() ? lw : lw * fast_exp2(mw - top);
  }
  const float factor = m == -__builtin_inff() ? 1.f : fast_exp2(m - top);
  const int64_t rows_all = g.batch * g.kv_heads * map.rows, base_row = (b * g.kv_heads + kvh) * (int64_t)map.rows;
  if (wave == 0 && h == 0 && there) {
    if (g.totals != nullptr) {
      float* st = g.stats + (split * rows_all + base_row + row) * 2;
      st[0] = top;
      st[1] = total;
    } else {
      g.lse[b * g.heads * (int64_t)r.t_q + map.at(row, r.t_q, 1)] = total == 0.f ? -__builtin_inff() : (top == -__builtin_inff() ? 0.f : top * ATT_LN2) + logf(total);
    }
  }
  const int orow = row0 + (threadIdx.x >> 3);
  float osum = 0.f;  // the total of the row this thread stores
  {
    __syncthreads();
    if (wave == 0 && h == 0) sm[n] = total;
    __syncthreads();
    osum = sm[threadIdx.x >> 3];
  }
  const float inv = osum == 0.f ? 0.f : 1.f / osum;
#pragma unroll
  for (int dt = 0; dt < DT; dt++) {
    const f32x4 x = gen_join(acc[dt], factor, lds);
    const int d = 32 * dt + (threadIdx.x & 7) * 4;
    if (orow < map.rows) {
      if (g.totals != nullptr) {
        float* o = g.totals + (split * rows_all + base_row + orow) * g.hd_v;
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (d + e < g.hd_v) o[d + e] = x[e];
      } else {
        S* o = (S*)g.out + b * g.heads * (int64_t)r.t_q * g.hd_v + map.at(orow, r.t_q, g.hd_v);
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (d + e < g.hd_v) T::store(o, d + e, osum == 0.f ? 0.f : x[e] * inv);
      }
    }
  }
  __syncthreads();
}

// ---- backward -------------------------------------------------------------------------------------------

struct GenBwd {
  const void* q;
  const void* k;
  const void* v;
  const void* out;
  const void* dout;
  const float* lse;
  float* delta;  // (batch, heads, t_q): rowsum(dout * out), written by the dQ pass
  void* dq;
  void* dk;
  void* dv;
  int heads, kv_heads, hd, hd_v, vec;
  float scale;
};

// dq of packed rows [row0, row0 + 32), and their delta.
template <typename T, int DT>
__device__ __forceinline__ void gen_dq_block(const GenBwd& g, const RuleArgs& ra, const RowMap& map, int64_t b, int kvh, int row0,
                                             bool write_delta, float* lds) {
  typedef typename T::Storage S;
  constexpr int CH = DT * 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const Rules r = rules_of(ra, b);
  const int row = row0 + n;
  const bool there = row < map.rows;
  const RowTile t = gen_row_tile(r, ra, map, row);
  const int64_t first = b * g.heads * (int64_t)r.t_q, here = there ? map.at(row, r.t_q, 1) : 0;
  const S* q = (const S*)g.q + (first + here) * g.hd;
  const S* o = (const S*)g.out + (first + here) * g.hd_v;
  const S* go = (const S*)g.dout + (first + here) * g.hd_v;
  const S* k = (const S*)g.k + (b * g.kv_heads + kvh) * (int64_t)r.t_k * g.hd;
  const S* v = (const S*)g.v + (b * g.kv_heads + kvh) * (int64_t)r.t_k * g.hd_v;

  f32x4 qf[CH], of[CH];
  f32x16 acc[DT];
  float delta = 0.f;
#pragma unroll
  for (int c = 0; c < CH; c++) {
    qf[c] = gen_load4<T>(q, there, 8 * c + 4 * h, g.hd, g.vec);
    of[c] = gen_load4<T>(go, there, 8 * c + 4 * h, g.hd_v, g.vec);
    const f32x4 x = gen_load4<T>(o, there, 8 * c + 4 * h, g.hd_v, g.vec);
#pragma unroll
    for (int e = 0; e < 4; e++) delta = fmaf(x[e], of[c][e], delta);
  }
#pragma unroll
  for (int dt = 0; dt < DT; dt++) acc[dt] = gen_zero();
  delta = gen_pair_sum(delta);
  if (write_delta && wave == 0 && h == 0 && there) g.delta[first + here] = delta;
  const float l2 = there ? att_l2(g.lse[first + here]) : __builtin_inff();

  int kend = r.len;
  if (r.causal) kend = min(kend, max(t.pmax + 1, r.pre));
  const int tiles = kend > 0 ? (kend + 31) / 32 : 0;
  for (int kt = wave; kt < tiles; kt += GEN_WAVES) {
    const int k0 = kt * 32;
    const int kd = gen_key_doc(r, k0 + n);
    if (gen_none(r, t, k0, kd)) continue;
    const bool whole = gen_whole(r, t, row0 + 32 <= map.rows, k0, kd), key_there = k0 + n < r.len;
    f32x16 s = gen_zero(), dp = gen_zero();
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const f32x4 a = gen_load4<T>(k + (int64_t)(k0 + n) * g.hd, key_there, 8 * c + 4 * h, g.hd, g.vec);
      const f32x4 w = gen_load4<T>(v + (int64_t)(k0 + n) * g.hd_v, key_there, 8 * c + 4 * h, g.hd_v, g.vec);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s = gen_mfma(a[e], qf[c][e], s);
        dp = gen_mfma(w[e], of[c][e], dp);
      }
    }
    unsigned vis = 0xffffu;
    float ds[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int at = 8 * (i >> 2) + 4 * h + (i & 3), key = k0 + at;
      float bent;
      const float y = gen_score(r, s[i], t.slope2, fabsf((float)(t.p - key)), bent);
      ds[i] = fast_exp2(y - l2) * (dp[i] - delta) * (g.scale * bent);
      if (!whole) {
        const int d = __shfl(kd, at);
        const bool see = there & sees(r, t.p, key) & (t.doc >= 0) & (d == t.doc);
        ds[i] = see ? ds[i] : 0.f;
        if (!see) vis &= ~(1u << i);
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
      float a[16];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int key = k0 + 8 * (i >> 2) + 4 * h + (i & 3);
        a[i] = gen_load1<T>(k + (int64_t)key * g.hd, key < r.len, 32 * dt + n, g.hd);
      }
      gen_add(acc[dt], a, ds, vis, !whole);
    }
  }
  const int orow = row0 + (threadIdx.x >> 3);
  S* dq = (S*)g.dq + (first + (orow < map.rows ? map.at(orow, r.t_q, 1) : 0)) * g.hd;
#pragma unroll
  for (int dt = 0; dt < DT; dt++) {
    const f32x4 x = gen_join(acc[dt], 1.f, lds);
    const int d = 32 * dt + (threadIdx.x & 7) * 4;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (orow < map.rows && d + e < g.hd) T::store(dq, d + e, x[e]);
  }
  __syncthreads();
}

// dk and dv of keys [key0, key0 + 32): a hidden key, one past the live ones too, gets zeros.
// KEEP: the resident fragments stay in registers; past 128 dims they would not fit beside the totals, and are read
// again for every tile (from L1).
template <typename T, int DT, bool KEEP = (DT <= 4)>
__device__ __forceinline__ void gen_dkv_block(const GenBwd& g, const RuleArgs& ra, const RowMap& map, int64_t b, int kvh, int key0,
                                              float* lds) {
  typedef typename T::Storage S;
  constexpr int CH = DT * 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const Rules r = rules_of(ra, b);
  const int key = key0 + n;
  const bool there = key < r.len;
  const int kd = gen_key_doc(r, key);
  const int64_t first = b * g.heads * (int64_t)r.t_q;
  const S* k = (const S*)g.k + ((b * g.kv_heads + kvh) * (int64_t)r.t_k + key) * g.hd;
  const S* v = (const S*)g.v + ((b * g.kv_heads + kvh) * (int64_t)r.t_k + key) * g.hd_v;
  const S* q = (const S*)g.q + first * g.hd;
  const S* go = (const S*)g.dout + first * g.hd_v;

  f32x4 kf[KEEP ? CH : 1], vf[KEEP ? CH : 1];
  if (KEEP) {
#pragma unroll
    for (int c = 0; c < CH; c++) {
      kf[KEEP ? c : 0] = gen_load4<T>(k, there, 8 * c + 4 * h, g.hd, g.vec);
      vf[KEEP ? c : 0] = gen_load4<T>(v, there, 8 * c + 4 * h, g.hd_v, g.vec);
    }
  }
  f32x16 gk[DT], gv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++) gk[dt] = gv[dt] = gen_zero();

  // the first row that can see one of the keys: query key0 - off, unless a prefix opens them to all. Of keys past the live
  // ones no row does, and key0 - off may be past t_q there, whose rows 32 bits do not count.
  const int tiles = key0 < r.len ? (map.rows + 31) / 32 : 0;
  int from = 0;
  if (tiles > 0 && r.causal && key0 >= r.pre) from = max(0, key0 - r.off) * map.group;
  for (int rt = from / 32 + wave; rt < tiles; rt += GEN_WAVES) {
    const int row0 = rt * 32, row = row0 + n;
    const bool row_there = row < map.rows;
    const RowTile t = gen_row_tile(r, ra, map, row);
    if (gen_none(r, t, key0, kd)) continue;
    const bool whole = gen_whole(r, t, row0 + 32 <= map.rows, key0, kd);
    const int64_t here = row_there ? map.at(row, r.t_q, 1) : 0;
    const float l2 = row_there ? att_l2(g.lse[first + here]) : __builtin_inff(), delta = row_there ? g.delta[first + here] : 0.f;
    f32x16 s = gen_zero(), dp = gen_zero();
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const f32x4 a = gen_load4<T>(q + here * g.hd, row_there, 8 * c + 4 * h, g.hd, g.vec);
      const f32x4 w = gen_load4<T>(go + here * g.hd_v, row_there, 8 * c + 4 * h, g.hd_v, g.vec);
      const f32x4 kc = KEEP ? kf[KEEP ? c : 0] : gen_load4<T>(k, there, 8 * c + 4 * h, g.hd, g.vec);
      const f32x4 vc = KEEP ? vf[KEEP ? c : 0] : gen_load4<T>(v, there, 8 * c + 4 * h, g.hd_v, g.vec);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s = gen_mfma(a[e], kc[e], s);
        dp = gen_mfma(w[e], vc[e], dp);
      }
    }
    unsigned vis = 0xffffu;
    float p[16], ds[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int at = 8 * (i >> 2) + 4 * h + (i & 3);
      const int pos = __shfl(t.p, at), d = __shfl(t.doc, at);
      const float li = __shfl(l2, at), de = __shfl(delta, at), sl = __shfl(t.slope2, at);
      float bent;
      const float y = gen_score(r, s[i], sl, fabsf((float)(pos - key)), bent);
      p[i] = fast_exp2(y - li);
      ds[i] = p[i] * (dp[i] - de) * (g.scale * bent);
      if (!whole) {
        const bool see = there & (row0 + at < map.rows) & sees(r, pos, key) & (d >= 0) & (d == kd);
        p[i] = see ? p[i] : 0.f;
        ds[i] = see ? ds[i] : 0.f;
        if (!see) vis &= ~(1u << i);
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
      float a[16], w[16];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int rr = row0 + 8 * (i >> 2) + 4 * h + (i & 3);
        const bool ok = rr < map.rows;
        const int64_t at = ok ? map.at(rr, r.t_q, 1) : 0;
        a[i] = gen_load1<T>(q + at * g.hd, ok, 32 * dt + n, g.hd);
        w[i] = gen_load1<T>(go + at * g.hd_v, ok, 32 * dt + n, g.hd_v);
      }
      gen_add(gk[dt], a, ds, vis, !whole);
      gen_add(gv[dt], w, p, vis, !whole);
    }
  }
  const int okey = key0 + (threadIdx.x >> 3);
  S* dk = (S*)g.dk + ((b * g.kv_heads + kvh) * (int64_t)r.t_k + okey) * g.hd;
  S* dv = (S*)g.dv + ((b * g.kv_heads + kvh) * (int64_t)r.t_k + okey) * g.hd_v;
#pragma unroll
  for (int dt = 0; dt < DT; dt++) {
    const int d = 32 * dt + (threadIdx.x & 7) * 4;
    const f32x4 x = gen_join(gk[dt], 1.f, lds), y = gen_join(gv[dt], 1.f, lds);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (okey < r.t_k && d + e < g.hd) T::store(dk, d + e, x[e]);
      if (okey < r.t_k && d + e < g.hd_v) T::store(dv, d + e, y[e]);
    }
  }
  __syncthreads();
}

}  // namespace
}  // namespace limn
