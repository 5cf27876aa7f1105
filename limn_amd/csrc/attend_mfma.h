// Attention with score rules on 16-bit matrix cores: bf16/f16 storage, float32 accumulation and statistics,
// hd == hd_v up to 128 in multiples of 8, run at a tile width D of 64, 96 or 128 (dims past hd are zeros).
//
// The decomposition and the orientation of the products are those of sdpa_mfma.h, whose tiles and LDS
// layout these kernels use: a workgroup of 4 waves owns 128 resident rows (queries of one head, or keys of one
// key head in the dK/dV pass), 32 a wave, one row a lane pair; the other side streams past in tiles of 64
// rows staged through LDS, consumed 32 at a time. What the rules add:
//  - tiles that no row of the block sees are not visited: past the last live key, past the diagonal (and the
//    prefix), or of documents whose range does not meet the block's (attend_ranges finds the range of every 32
//    positions first; a block turns them into one bit a tile in LDS);
//  - a half tile that every row of the wave sees whole takes no element tests (a wave-uniform branch);
//  - the cap and the distance are float arithmetic on the score tile. Per 32 x 32 tile at D = 128 the matrix
//    cores take 512 cycles a wave for the forward's two products; the softmax takes 16 exponentials of 16
//    cycles and about 6 other operations of 4 an element, the cap an exponential and a reciprocal more,
//    so capped attention is bound by the vector ALU.
//  - the query heads of a key head are one loop of the dK/dV pass: their gradients are one sum in head order.
//
// Hidden pairs have exact zeros in the second products, but a zero times an infinity or a NaN is NaN. Such a
// result stays NaN to the end of the block, so a block whose totals are not all finite says so (odd), and a
// launch behind the pass computes those blocks again in float arithmetic (attend_mend.hip, by attend_general.h's
// blocks, which leave hidden pairs out whatever they hold). Nothing in the loops pays for it; with the float
// blocks in the same kernel their registers halved the occupancy and spilled the loops' own.
#pragma once

#include "attend_fast.h"
#include "sdpa_mfma.h"

namespace limn {
namespace {

constexpr int ATT_WORDS = 32;      // 64-tile words of the visit list: 131072 streamed rows
constexpr int ATT_MOST_DOC_KEYS = ATT_WORDS * 64 * TILE;

// ---- documents: ranges, visit lists ---------------------------------------------------------------------

struct DocRange {
  int lo, hi;
  bool part;  // some positions have no document
  __device__ __forceinline__ bool meets(const DocRange& o) const { return lo <= hi && o.lo <= o.hi && lo <= o.hi && o.lo <= hi; }
  __device__ __forceinline__ bool is(int doc) const { return !part && lo == doc && hi == doc; }
};

// positions [p0, p1], which may reach outside [0, 32 granules)
__device__ __forceinline__ DocRange doc_range(const int2* ranges, int granules, int p0, int p1) {
  DocRange r = {0x7fffffff, 0, p0 < 0 || p1 >= granules * 32};
  const int g0 = max(p0, 0) >> 5, g1 = min(p1 >> 5, granules - 1);
  for (int g = g0; g <= g1; g++) {
    const int2 e = ranges[g];
    r.lo = min(r.lo, e.x);
    r.hi = max(r.hi, e.y & 0x7fffffff);
    r.part |= e.y < 0;
  }
  return r;
}

// The streamed tiles a block visits, in order: [from, to), or those with a bit set.
struct Visit {
  int to;
  const uint64_t* bits;  // LDS, or nullptr: every tile
  __device__ __forceinline__ int next(int t) const {
    if (bits == nullptr || t >= to) return t;
    int w = t >> 6;
    uint64_t m = bits[w] >> (t & 63);
    while (m == 0) {
      if (++w * 64 >= to) return to;
      t = w * 64;
      m = bits[w];
    }
    t += __builtin_ctzll(m);
    return __builtin_amdgcn_readfirstlane(t < to ? t : to);
  }
};

// ---- rows of hd elements in tiles of D ------------------------------------------------------------------

struct HeadRows {
  __amdgpu_buffer_rsrc_t rsrc;
  int hd;
  __device__ __forceinline__ HeadRows(const u16* base, int rows, int hd_) : hd(hd_) {
    rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, rows * hd_ * 2, 0x00020000);
  }
  // elements [d, d + 8) of a row: zeros past the rows and past hd
  __device__ __forceinline__ u16x8 load8(int row, int d) const {
    const int off = d < hd ? (row * hd + d) * 2 : 0x7ffffff0;
    return __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0));
  }
};

// Global -> registers -> LDS staging of two 64-row tiles, as Stage<D> of sdpa_mfma.h does it.
template <int D>
struct HeadStage {
  static constexpr int COLS = D / 8, PER_TILE = COLS * (TILE / 4), SLOTS = (2 * PER_TILE + THREADS - 1) / THREADS;
  u16x8 r[SLOTS][4];
  __device__ __forceinline__ void load(const HeadRows& m0, const HeadRows& m1, int row0) {
#pragma unroll
    for (int s = 0; s < SLOTS; s++) {
      const int idx = threadIdx.x + s * THREADS;
      if (idx < 2 * PER_TILE) {
        const int which = __builtin_amdgcn_readfirstlane(idx / PER_TILE), w = idx - which * PER_TILE;
        const int col = w % COLS, grp = w / COLS;
        const HeadRows& m = which ? m1 : m0;
#pragma unroll
        for (int e = 0; e < 4; e++) r[s][e] = m.load8(row0 + grp * 4 + e, col * 8);
      }
    }
  }
  __device__ __forceinline__ void store(u16* tile0, u16* tile1) {
#pragma unroll
    for (int s = 0; s < SLOTS; s++) {
      const int idx = threadIdx.x + s * THREADS;
      if (idx < 2 * PER_TILE) {
        const int which = idx / PER_TILE, w = idx - which * PER_TILE;
        const int col = w % COLS, grp = w / COLS;
        u16* tile = which ? tile1 : tile0;
#pragma unroll
        for (int e = 0; e < 4; e++) *(u16x8*)(tile + tile_at<D>(grp * 4 + e, col * 8)) = r[s][e];
      }
    }
  }
};

// store_staged of sdpa_mfma.h for rows of hd elements
template <typename T, int D>
__device__ __forceinline__ void store_rows(u16* base, const f32x16* acc, int row0, int rows, int hd, float mul, u16* stage) {
  const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31;
  constexpr int RS = D + 8, CPR = D / 8;
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const u16x4 o = {T::pack(acc[dt][4 * g] * mul), T::pack(acc[dt][4 * g + 1] * mul), T::pack(acc[dt][4 * g + 2] * mul),
                       T::pack(acc[dt][4 * g + 3] * mul)};
      *(u16x4*)(stage + n * RS + dt * 32 + 8 * g + 4 * h) = o;
    }
#pragma unroll
  for (int j = 0; j < 32 * CPR / 64; j++) {
    const int r = (j * 64 + lane) / CPR, c = (j * 64 + lane) % CPR;
    const u16x8 v = *(const u16x8*)(stage + r * RS + c * 8);
    if (row0 + r < rows && c * 8 < hd) *(u16x8*)(base + (int64_t)(row0 + r) * hd + c * 8) = v;
  }
}

// Whether any of the workgroup's totals is not finite.
template <int N>
__device__ __forceinline__ bool any_odd(const f32x16 (&acc)[N]) {
  float x = 0.f;  // a finite number times 0 stays 0
#pragma unroll
  for (int dt = 0; dt < N; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) x = fmaf(acc[dt][i], 0.f, x);
  return __syncthreads_or(x != 0.f);
}

// float16 has no normal numbers below 2^-14: probabilities go into its products multiplied by a power of two, 2^7
// in the forward (where the reference point lets them reach 2^8) and 2^14 in the dV product (where none
// passes 1), taken off again at the store. bfloat16 has float32's range.
template <typename T>
constexpr float shift_of(float bits) {
  return std::is_same<T, F16>::value ? bits : 0.f;
}

// ---- scores ---------------------------------------------------------------------------------------------

// A score tile item into log2 units (as it is, if there is neither cap nor distance: then c2 comes in with
// the exponential), and for the backward the cap's derivative.
template <bool CAP, bool BIAS, bool GRAD>
__device__ __forceinline__ float bend(float x, const Rules& r, float slope2, float far, float& bent) {
  float y = x;
  if (CAP) {
    // tanh(z) = 1 - 2 / (1 + e^2z): off by some 2^-23 absolutely, a part of a half width's step after the
    // softmax; the derivative 1 - tanh^2 = 4 w (1 - w) with w = 1 / (1 + e^2z)
    const float w = __builtin_amdgcn_rcpf(1.f + fast_exp2(x * r.cap_in));
    y = fmaf(-2.f * r.cap_out, w, r.cap_out);
    if (GRAD) bent = 4.f * w * (1.f - w);
  } else if (BIAS) {
    y = x * r.c2;
  }
  if (BIAS) y = fmaf(-slope2, fabsf(far), y);
  return y;
}

// ---- forward --------------------------------------------------------------------------------------------

template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 2) void attend_fwd_mfma(FastArgs g, RuleArgs ra) {
  constexpr int TE = TILE * tile_stride<D>();
  constexpr bool RAW = !CAP && !BIAS;
  constexpr float UP = shift_of<T>(7.f);
  __shared__ __attribute__((aligned(16))) u16 tiles[4 * TE];
  __shared__ __attribute__((aligned(16))) int kdocs[2][TILE];
  __shared__ uint64_t bits[ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const int64_t nqb = (ra.t_q + ATT_ROWS - 1) / ATT_ROWS;
  int64_t bh, blk;
  head_and_block(g.batch * g.heads, nqb, bh, blk);
  const int64_t b = bh / g.heads;
  const int head = (int)(bh - b * g.heads), kvh = head / (g.heads / g.kv_heads);
  const int q0 = (int)(nqb - 1 - blk) * ATT_ROWS, wq0 = q0 + wave * 32, row = wq0 + n;  // causal: the longest rows go first
  const Rules r = rules_of(ra, b);
  const int p = r.off + row;
  const bool there = row < r.t_q;
  const int doc = there ? query_doc(r, p) : -1;
  const float slope2 = BIAS ? ra.slopes[head] * LOG2E : 0.f;
  const HeadRows qrows(g.q + bh * (int64_t)r.t_q * g.hd, r.t_q, g.hd);
  const int64_t kv = (b * g.kv_heads + kvh) * (int64_t)r.t_k * g.hd;
  const HeadRows krows(g.k + kv, r.len, g.hd), vrows(g.v + kv, r.len, g.hd);  // keys past the live ones read as zeros
  const float unit = RAW ? r.c2 : 1.f, lift = RESCALE_LOG2 / unit;

  u16x8 qf[D / 16];
  f32x16 acc[D / 32];
  float m = neg_inf(), l = 0.f;
#pragma unroll
  for (int ds = 0; ds < D / 16; ds++) qf[ds] = qrows.load8(row, ds * 16 + 8 * h);
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++) acc[dt] = zero16();

  const int last = min(q0 + ATT_ROWS, r.t_q) - 1;  // the block's last query
  int kend = r.len;
  if (r.causal) kend = min(kend, max(r.off + last + 1, r.pre));
  Visit visit = {kend > 0 ? (kend + TILE - 1) / TILE : 0, nullptr};
  const int2* ranges = g.ranges ? g.ranges + b * g.granules : nullptr;
  int wave_doc = 0;  // the document of every row of the wave, or -1
  if (ranges != nullptr) {
    const DocRange mine = doc_range(ranges, g.granules, r.off + q0, r.off + last);
    for (int w = wave; w * 64 < visit.to; w += WAVES) {
      const int t = w * 64 + lane;
      const bool meets = t < visit.to && mine.meets(doc_range(ranges, g.granules, t * TILE, min(t * TILE + TILE, g.granules * 32) - 1));
      const uint64_t word = __ballot(meets);
      if (lane == 0) bits[w] = word;
    }
    visit.bits = bits;
    const int first = __builtin_amdgcn_readfirstlane(doc);
    wave_doc = __all(doc == first) ? first : -1;
    __syncthreads();
  }

  HeadStage<D> st;
  int dnext = 0;
  int cur = visit.next(0), nxt = cur < visit.to ? visit.next(cur + 1) : visit.to;
  auto docs_load = [&](int t) { return ranges != nullptr && threadIdx.x < TILE && t * TILE + (int)threadIdx.x < r.len ? r.docs[t * TILE + threadIdx.x] : -1; };
  if (cur < visit.to) {
    st.load(krows, vrows, cur * TILE);
    dnext = docs_load(cur);
    st.store(tiles, tiles + TE);
    if (threadIdx.x < TILE) kdocs[0][threadIdx.x] = dnext;
    if (nxt < visit.to) {
      st.load(krows, vrows, nxt * TILE);
      dnext = docs_load(nxt);
    }
  }
  __syncthreads();
  for (int buf = 0; cur < visit.to; buf ^= 1) {
    const int k0 = cur * TILE;
    const u16* Kt = tiles + 2 * buf * TE;
    const u16* Vt = Kt + TE;
#pragma unroll
    for (int sub = 0; sub < 2; sub++) {
      const int s0 = k0 + sub * 32;
      u16x8 kfr[D / 16];
#pragma unroll
      for (int ds = 0; ds < D / 16; ds++) kfr[ds] = read_row<D>(Kt, sub * 32 + n, 2 * ds + h);
      f32x16 s = zero16();
#pragma unroll
      for (int ds = 0; ds < D / 16; ds++) s = T::mfma32(kfr[ds], qf[ds], s);
      const float near = (float)(p - s0 - 4 * h);
      if (!RAW) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float unused;
          s[i] = bend<CAP, BIAS, false>(s[i], r, slope2, near - (float)(8 * (i >> 2) + (i & 3)), unused);
        }
      }
      bool edge = s0 + 32 > r.len || (r.causal && s0 + 31 > r.off + wq0 && s0 + 31 >= r.pre);
      if (ranges != nullptr && !edge) {
        const int2 e = ranges[s0 >> 5];
        edge = wave_doc < 0 || e.x != wave_doc || e.y != wave_doc;
      }
      if (edge) {
        if (ranges != nullptr) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int4 d4 = *(const int4*)&kdocs[buf][sub * 32 + 8 * q + 4 * h];
            const int dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
            for (int e = 0; e < 4; e++) s[4 * q + e] = (doc >= 0) & (dd[e] == doc) ? s[4 * q + e] : neg_inf();
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = sees(r, p, s0 + 8 * (i >> 2) + 4 * h + (i & 3)) ? s[i] : neg_inf();
      }
      float mx = neg_inf();
#pragma unroll
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[i]);
      mx = pair_max(mx);
      if (__any(mx > m + lift)) {  // the reference point moves rarely: see sdpa_fwd_mfma
        const float mnew = fmaxf(m, mx);
        const float alpha = mnew == neg_inf() ? 1.f : fast_exp2((m - mnew) * unit);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++) acc[dt] *= alpha;
        m = mnew;
      }
      const float base = (m == neg_inf() ? 0.f : m * unit) - UP;
      float rs = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float e = RAW ? fast_exp2(fmaf(s[i], unit, -base)) : fast_exp2(s[i] - base);
        s[i] = e;
        rs += e;
      }
      l += rs;
#pragma unroll
      for (int c = 0; c < 2; c++) {
        u16x8 vfr[D / 32];
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++) vfr[dt] = read_transposed<D>(Vt, sub * 32 + 16 * c, dt * 32);
        const u16x8 pb = pack8<T>(s, 8 * c);
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++) acc[dt] = T::mfma32(vfr[dt], pb, acc[dt]);
      }
    }
    cur = nxt;
    if (cur < visit.to) {
      u16* Kn = tiles + 2 * (buf ^ 1) * TE;
      st.store(Kn, Kn + TE);
      if (threadIdx.x < TILE) kdocs[buf ^ 1][threadIdx.x] = dnext;
      nxt = visit.next(cur + 1);
      if (nxt < visit.to) {
        st.load(krows, vrows, nxt * TILE);
        dnext = docs_load(nxt);
      }
    }
    __syncthreads();
  }
  const float total = pair_sum(l);
  const bool odd = any_odd(acc);
  if (threadIdx.x == 0) g.odd[bh * nqb + q0 / ATT_ROWS] = odd;
  const float inv = total == 0.f ? 0.f : 1.f / total;  // a row that sees nothing is a row of zeros
  store_rows<T, D>(g.o0 + bh * (int64_t)r.t_q * g.hd, acc, wq0, r.t_q, g.hd, inv, tiles + wave * TE);
  if (h == 0 && there) g.lse[bh * (int64_t)r.t_q + row] = total == 0.f ? neg_inf() : (m * unit - UP) * ATT_LN2 + logf(total);
}

// ---- dQ pass: also delta = rowsum(dout * out), which the dK/dV pass reads ---------------------------------

template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 2) void attend_dq_mfma(FastArgs g, RuleArgs ra) {
  constexpr int TE = TILE * tile_stride<D>();
  constexpr bool RAW = !CAP && !BIAS;
  __shared__ __attribute__((aligned(16))) u16 tiles[4 * TE];
  __shared__ __attribute__((aligned(16))) int kdocs[2][TILE];
  __shared__ uint64_t bits[ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const int64_t nqb = (ra.t_q + ATT_ROWS - 1) / ATT_ROWS;
  int64_t bh, blk;
  head_and_block(g.batch * g.heads, nqb, bh, blk);
  const int64_t b = bh / g.heads;
  const int head = (int)(bh - b * g.heads), kvh = head / (g.heads / g.kv_heads);
  const int q0 = (int)(nqb - 1 - blk) * ATT_ROWS, wq0 = q0 + wave * 32, row = wq0 + n;
  const Rules r = rules_of(ra, b);
  const int p = r.off + row;
  const bool there = row < r.t_q;
  const int doc = there ? query_doc(r, p) : -1;
  const float slope2 = BIAS ? ra.slopes[head] * LOG2E : 0.f;
  const int64_t rows0 = bh * (int64_t)r.t_q;
  const HeadRows qrows(g.q + rows0 * g.hd, r.t_q, g.hd), grows(g.dout + rows0 * g.hd, r.t_q, g.hd), orows(g.out + rows0 * g.hd, r.t_q, g.hd);
  const int64_t kv = (b * g.kv_heads + kvh) * (int64_t)r.t_k * g.hd;
  const HeadRows krows(g.k + kv, r.len, g.hd), vrows(g.v + kv, r.len, g.hd);

  u16x8 qf[D / 16], of[D / 16];
  f32x16 acc[D / 32];
  float delta = 0.f;
#pragma unroll
  for (int ds = 0; ds < D / 16; ds++) {
    qf[ds] = qrows.load8(row, ds * 16 + 8 * h);
    of[ds] = grows.load8(row, ds * 16 + 8 * h);
    const u16x8 o = orows.load8(row, ds * 16 + 8 * h);
#pragma unroll
    for (int e = 0; e < 8; e++) delta = fmaf(T::unpack(of[ds][e]), T::unpack(o[e]), delta);
  }
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++) acc[dt] = zero16();
  delta = pair_sum(delta);
  if (h == 0 && there) g.delta[rows0 + row] = delta;
  const float l2 = there ? att_l2(g.lse_in[rows0 + row]) : __builtin_inff();

  const int last = min(q0 + ATT_ROWS, r.t_q) - 1;
  int kend = r.len;
  if (r.causal) kend = min(kend, max(r.off + last + 1, r.pre));
  Visit visit = {kend > 0 ? (kend + TILE - 1) / TILE : 0, nullptr};
  const int2* ranges = g.ranges ? g.ranges + b * g.granules : nullptr;
  int wave_doc = 0;
  if (ranges != nullptr) {
    const DocRange mine = doc_range(ranges, g.granules, r.off + q0, r.off + last);
    for (int w = wave; w * 64 < visit.to; w += WAVES) {
      const int t = w * 64 + lane;
      const bool meets = t < visit.to && mine.meets(doc_range(ranges, g.granules, t * TILE, min(t * TILE + TILE, g.granules * 32) - 1));
      const uint64_t word = __ballot(meets);
      if (lane == 0) bits[w] = word;
    }
    visit.bits = bits;
    const int first = __builtin_amdgcn_readfirstlane(doc);
    wave_doc = __all(doc == first) ? first : -1;
    __syncthreads();
  }

  HeadStage<D> st;
  int dnext = 0;
  int cur = visit.next(0), nxt = cur < visit.to ? visit.next(cur + 1) : visit.to;
  auto docs_load = [&](int t) { return ranges != nullptr && threadIdx.x < TILE && t * TILE + (int)threadIdx.x < r.len ? r.docs[t * TILE + threadIdx.x] : -1; };
  if (cur < visit.to) {
    st.load(krows, vrows, cur * TILE);
    dnext = docs_load(cur);
    st.store(tiles, tiles + TE);
    if (threadIdx.x < TILE) kdocs[0][threadIdx.x] = dnext;
    if (nxt < visit.to) {
      st.load(krows, vrows, nxt * TILE);
      dnext = docs_load(nxt);
    }
  }
  __syncthreads();
  for (int buf = 0; cur < visit.to; buf ^= 1) {
    const int k0 = cur * TILE;
    const u16* Kt = tiles + 2 * buf * TE;
    const u16* Vt = Kt + TE;
#pragma unroll
    for (int sub = 0; sub < 2; sub++) {
      const int s0 = k0 + sub * 32;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ds = 0; ds < D / 16; ds++) {
        s = T::mfma32(read_row<D>(Kt, sub * 32 + n, 2 * ds + h), qf[ds], s);
        dp = T::mfma32(read_row<D>(Vt, sub * 32 + n, 2 * ds + h), of[ds], dp);
      }
      const float near = (float)(p - s0 - 4 * h);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float bent = 1.f;
        const float y = bend<CAP, BIAS, true>(s[i], r, slope2, near - (float)(8 * (i >> 2) + (i & 3)), bent);
        const float e = fast_exp2(RAW ? fmaf(y, r.c2, -l2) : y - l2);
        s[i] = e * (dp[i] - delta) * (CAP ? bent : 1.f);  // times scale once, at the store
      }
      bool edge = s0 + 32 > r.len || (r.causal && s0 + 31 > r.off + wq0 && s0 + 31 >= r.pre);
      if (ranges != nullptr && !edge) {
        const int2 e = ranges[s0 >> 5];
        edge = wave_doc < 0 || e.x != wave_doc || e.y != wave_doc;
      }
      if (edge) {
        if (ranges != nullptr) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int4 d4 = *(const int4*)&kdocs[buf][sub * 32 + 8 * q + 4 * h];
            const int dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
            for (int e = 0; e < 4; e++) s[4 * q + e] = (doc >= 0) & (dd[e] == doc) ? s[4 * q + e] : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = sees(r, p, s0 + 8 * (i >> 2) + 4 * h + (i & 3)) ? s[i] : 0.f;
      }
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const u16x8 gb = pack8<T>(s, 8 * c);
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++) acc[dt] = T::mfma32(read_transposed<D>(Kt, sub * 32 + 16 * c, dt * 32), gb, acc[dt]);
      }
    }
    cur = nxt;
    if (cur < visit.to) {
      u16* Kn = tiles + 2 * (buf ^ 1) * TE;
      st.store(Kn, Kn + TE);
      if (threadIdx.x < TILE) kdocs[buf ^ 1][threadIdx.x] = dnext;
      nxt = visit.next(cur + 1);
      if (nxt < visit.to) {
        st.load(krows, vrows, nxt * TILE);
        dnext = docs_load(nxt);
      }
    }
    __syncthreads();
  }
  const bool odd = any_odd(acc);
  if (threadIdx.x == 0) g.odd[bh * nqb + q0 / ATT_ROWS] = odd;
  store_rows<T, D>(g.o0 + rows0 * g.hd, acc, wq0, r.t_q, g.hd, g.scale, tiles + wave * TE);
}

// ---- dK/dV pass -----------------------------------------------------------------------------------------

template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, D <= 64 ? 2 : 1) void attend_dkv_mfma(FastArgs g, RuleArgs ra) {
  constexpr int TE = TILE * tile_stride<D>();
  constexpr bool RAW = !CAP && !BIAS;
  constexpr float UP = shift_of<T>(14.f), DOWN = std::is_same<T, F16>::value ? 1.f / 16384.f : 1.f;
  __shared__ __attribute__((aligned(16))) u16 tiles[4 * TE];
  __shared__ __attribute__((aligned(16))) float Ls[2][TILE];
  __shared__ __attribute__((aligned(16))) float Ds[2][TILE];
  __shared__ __attribute__((aligned(16))) int qdocs[2][TILE];
  __shared__ uint64_t bits[ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const int64_t nkb = (ra.t_k + ATT_ROWS - 1) / ATT_ROWS;
  int64_t bk, blk;
  head_and_block(g.batch * g.kv_heads, nkb, bk, blk);  // causal: the first keys are seen by the most queries
  const int64_t b = bk / g.kv_heads;
  const int kvh = (int)(bk - b * g.kv_heads), group = g.heads / g.kv_heads;
  const int k0 = (int)blk * ATT_ROWS, wk0 = k0 + wave * 32, key = wk0 + n;
  const Rules r = rules_of(ra, b);
  const bool there = key < r.len;
  const int doc = r.docs != nullptr ? (there ? r.docs[key] : -1) : 0;
  const HeadRows krows(g.k + bk * (int64_t)r.t_k * g.hd, r.len, g.hd), vrows(g.v + bk * (int64_t)r.t_k * g.hd, r.len, g.hd);

  u16x8 kf[D / 16], vf[D / 16];
  f32x16 gk[D / 32], gv[D / 32];
#pragma unroll
  for (int ds = 0; ds < D / 16; ds++) {
    kf[ds] = krows.load8(key, ds * 16 + 8 * h);
    vf[ds] = vrows.load8(key, ds * 16 + 8 * h);
  }
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++) gk[dt] = gv[dt] = zero16();

  // query tiles: from the first that can see the block's first key on, unless a prefix opens it to all
  const int first_q = r.causal && k0 >= r.pre ? max(0, k0 - r.off) / TILE : 0;
  Visit visit = {k0 < r.len ? (r.t_q + TILE - 1) / TILE : 0, nullptr};
  const int2* ranges = g.ranges ? g.ranges + b * g.granules : nullptr;
  int wave_doc = 0;
  if (ranges != nullptr) {
    const DocRange mine = doc_range(ranges, g.granules, k0, min(k0 + ATT_ROWS, r.t_k) - 1);
    for (int w = wave; w * 64 < visit.to; w += WAVES) {
      const int t = w * 64 + lane;
      const bool meets = t < visit.to && mine.meets(doc_range(ranges, g.granules, r.off + t * TILE, r.off + min(t * TILE + TILE, r.t_q) - 1));
      const uint64_t word = __ballot(meets);
      if (lane == 0) bits[w] = word;
    }
    visit.bits = bits;
    const int first = __builtin_amdgcn_readfirstlane(doc);
    wave_doc = __all(doc == first) ? first : -1;
    __syncthreads();
  }

  HeadStage<D> st;
  float lnext = 0.f, dnext = 0.f;
  int qnext = -1;
  const int64_t head_rows = r.t_q;
  const int64_t base_row = (b * g.heads + kvh * (int64_t)group) * head_rows;
  // tile `t` of query head `gh` of the group
  auto load = [&](int gh, int t) __attribute__((always_inline)) {
    const int64_t rows0 = base_row + gh * head_rows;
    const HeadRows qrows(g.q + rows0 * g.hd, r.t_q, g.hd), grows(g.dout + rows0 * g.hd, r.t_q, g.hd);
    st.load(qrows, grows, t * TILE);
    if (threadIdx.x < TILE) {
      const int qq = t * TILE + (int)threadIdx.x;
      const bool ok = qq < r.t_q;
      lnext = ok ? att_l2(g.lse_in[rows0 + qq]) - UP : __builtin_inff();
      dnext = ok ? g.delta[rows0 + qq] * DOWN : 0.f;
      qnext = ok ? query_doc(r, r.off + qq) : -1;
    }
  };
  auto store = [&](int buf) __attribute__((always_inline)) {
    u16* Qn = tiles + 2 * buf * TE;
    st.store(Qn, Qn + TE);
    if (threadIdx.x < TILE) {
      Ls[buf][threadIdx.x] = lnext;
      Ds[buf][threadIdx.x] = dnext;
      qdocs[buf][threadIdx.x] = qnext;
    }
  };
  const int begin = visit.next(first_q);
  int gh = 0, cur = begin, ngh = 0, nxt = begin;
  // the tile after (ngh, nxt): the head's next, or the next head's first
  auto advance = [&]() __attribute__((always_inline)) {
    nxt = visit.next(nxt + 1);
    if (nxt >= visit.to) {
      ngh++;
      nxt = begin;
    }
  };
  const bool any = begin < visit.to;
  if (any) {
    load(gh, cur);
    store(0);
    advance();
    if (ngh < group) load(ngh, nxt);
  }
  __syncthreads();
  for (int buf = 0; any && gh < group; buf ^= 1) {
    const int r0 = cur * TILE;
    const float slope2 = BIAS ? ra.slopes[kvh * group + gh] * LOG2E : 0.f;
    const u16* Qt = tiles + 2 * buf * TE;
    const u16* Gt = Qt + TE;
#pragma unroll
    for (int sub = 0; sub < 2; sub++) {
      const int s0 = r0 + sub * 32;
      f32x16 s = zero16(), dp = zero16();
      u16x8 qa[D / 16], ga[D / 16];
#pragma unroll
      for (int ds = 0; ds < D / 16; ds++) {
        qa[ds] = read_row<D>(Qt, sub * 32 + n, 2 * ds + h);
        ga[ds] = read_row<D>(Gt, sub * 32 + n, 2 * ds + h);
      }
#pragma unroll
      for (int ds = 0; ds < D / 16; ds++) {
        s = T::mfma32(qa[ds], kf[ds], s);
        dp = T::mfma32(ga[ds], vf[ds], dp);
      }
      f32x4 l4[4], d4[4];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        l4[q] = *(const f32x4*)&Ls[buf][sub * 32 + 8 * q + 4 * h];
        d4[q] = *(const f32x4*)&Ds[buf][sub * 32 + 8 * q + 4 * h];
      }
      const float near = (float)(r.off + s0 + 4 * h - key);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float bent = 1.f;
        const float y = bend<CAP, BIAS, true>(s[i], r, slope2, near + (float)(8 * (i >> 2) + (i & 3)), bent);
        const float l2 = l4[i >> 2][i & 3];
        s[i] = fast_exp2(RAW ? fmaf(y, r.c2, -l2) : y - l2);
        dp[i] = s[i] * fmaf(dp[i], DOWN, -d4[i >> 2][i & 3]) * (CAP ? bent : 1.f);  // times scale once, at the store
      }
      bool edge = s0 + 32 > r.t_q || wk0 + 32 > r.len || (r.causal && r.off + s0 < wk0 + 31 && wk0 + 31 >= r.pre);
      if (ranges != nullptr && !edge) edge = wave_doc < 0 || !doc_range(ranges, g.granules, r.off + s0, r.off + s0 + 31).is(wave_doc);
      if (edge) {
        if (ranges != nullptr) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int4 q4 = *(const int4*)&qdocs[buf][sub * 32 + 8 * q + 4 * h];
            const int dd[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const bool same = (doc >= 0) & (dd[e] == doc);
              s[4 * q + e] = same ? s[4 * q + e] : 0.f;
              dp[4 * q + e] = same ? dp[4 * q + e] : 0.f;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int qq = s0 + 8 * (i >> 2) + 4 * h + (i & 3);
          const bool see = (qq < r.t_q) & sees(r, r.off + qq, key);
          s[i] = see ? s[i] : 0.f;
          dp[i] = see ? dp[i] : 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const u16x8 pb = pack8<T>(s, 8 * c), gb = pack8<T>(dp, 8 * c);
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++) {
          gv[dt] = T::mfma32(read_transposed<D>(Gt, sub * 32 + 16 * c, dt * 32), pb, gv[dt]);
          gk[dt] = T::mfma32(read_transposed<D>(Qt, sub * 32 + 16 * c, dt * 32), gb, gk[dt]);
        }
      }
    }
    gh = ngh;
    cur = nxt;
    if (gh < group) {
      store(buf ^ 1);
      advance();
      if (ngh < group) load(ngh, nxt);
    }
    __syncthreads();
  }
  const bool odd_k = any_odd(gk), odd_v = any_odd(gv);
  if (threadIdx.x == 0) g.odd[bk * nkb + blk] = odd_k | odd_v;
  store_rows<T, D>(g.o0 + bk * (int64_t)r.t_k * g.hd, gk, wk0, r.t_k, g.hd, g.scale, tiles + wave * TE);
  store_rows<T, D>(g.o1 + bk * (int64_t)r.t_k * g.hd, gv, wk0, r.t_k, g.hd, DOWN, tiles + wave * TE);
}

// ---- launches -------------------------------------------------------------------------------------------

enum AttendPass { ATTEND_PASS_FWD, ATTEND_PASS_DQ, ATTEND_PASS_DKV };

template <AttendPass PASS, typename T, int D, bool CAP, bool BIAS>
int launch_fast_as(const FastArgs& g, const RuleArgs& ra, hipStream_t stream) {
  const int64_t blocks = PASS == ATTEND_PASS_DKV ? g.batch * g.kv_heads * ((ra.t_k + ATT_ROWS - 1) / ATT_ROWS)
                                                 : g.batch * g.heads * ((ra.t_q + ATT_ROWS - 1) / ATT_ROWS);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "attend: %lld workgroups exceed one launch", (long long)blocks);
  const dim3 grid((unsigned)blocks), block(THREADS);
  if constexpr (PASS == ATTEND_PASS_FWD)
    hipLaunchKernelGGL((attend_fwd_mfma<T, D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  else if constexpr (PASS == ATTEND_PASS_DQ)
    hipLaunchKernelGGL((attend_dq_mfma<T, D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  else
    hipLaunchKernelGGL((attend_dkv_mfma<T, D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  return check_hip(hipGetLastError(), "launching attention");
}

template <AttendPass PASS, typename T, int D>
int launch_fast_rules(const FastArgs& g, const RuleArgs& ra, hipStream_t stream) {
  const bool cap = ra.softcap > 0.f, bias = ra.slopes != nullptr;
  if (cap) return bias ? launch_fast_as<PASS, T, D, true, true>(g, ra, stream) : launch_fast_as<PASS, T, D, true, false>(g, ra, stream);
  return bias ? launch_fast_as<PASS, T, D, false, true>(g, ra, stream) : launch_fast_as<PASS, T, D, false, false>(g, ra, stream);
}

}  // namespace
}  // namespace limn
