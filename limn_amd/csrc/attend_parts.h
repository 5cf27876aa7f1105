// Attention with score rules for float32 on bf16 matrix cores: every operand as the sum of three bf16 numbers,
// x = h + m + l (h the nearest to x, m to x - h, l to the rest: x to 2^-24 or better, down to half of bf16's least step,
// 2^-134), every product of two as the six products of parts that are not below 2^-24 of it (the splitting
// published as BF16x6: Henry, Tang, Heinecke, Leveraging the bfloat16 artificial intelligence datatype for
// higher-precision computations, 2019). The five small ones are summed apart from h h, so that the
// rounding of the total's sum is that of one float32 product each. Six products at the 16-bit rate are 2.6 times
// as fast as one at the float32 matrix rate.
//
// The passes, orientation and visit lists are those of the half widths up to 64 dims (attend_mfma.h): a workgroup
// of 4 waves owns 128 resident rows whose parts sit in registers; the other side streams past in tiles of 64 rows (32
// past 64 dims), loaded as float a tile ahead and split on the way into LDS, six matrices of a tile at a time
// (52 to 55 KB), where the waves share them: the general kernels, whose waves each read a tile of their own for
// 32 resident rows, are bound by those reads (27 of 157 TFLOP/s).
//
// Caps take cap_scores' exact form: 8 x 16 heads x 1024 x 64 under a cap of 50 forward 141 us and backward 548, where the short
// form of the half widths took 138 and 515 and lost 4 bits.
//
// A total that is not finite, also where a finite operand is past bf16's largest number, has its block computed again in
// float (attend_mend.hip).
#pragma once

#include "attend_mfma.h"

namespace limn {
namespace {

template <int D>
struct PartTile {
  static constexpr int ROWS = D <= 64 ? 64 : 32, SUBS = ROWS / 32;
  static constexpr int MATRIX = ROWS * tile_stride<D>();  // elements of one part
};

struct Parts8 {
  u16x8 p[3];
};

__device__ __forceinline__ Parts8 split8(const float* v) {
  Parts8 o;
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = v[e];
#pragma unroll
  for (int part = 0; part < 3; part++) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      w[e] = BF16::pack2(r[2 * e], r[2 * e + 1]);
      if (part < 2) {
        r[2 * e] -= __uint_as_float(w[e] << 16);
        r[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
      }
    }
    o.p[part] = __builtin_bit_cast(u16x8, w);
  }
  return o;
}
// items base .. base + 7 of an accumulator: a B operand, as pack8
__device__ __forceinline__ Parts8 split_items(const f32x16& s, int base) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = s[base + e];
  return split8(v);
}

// big += h h, small += the other five, the smallest first
__device__ __forceinline__ void six(const Parts8& a, const Parts8& b, f32x16& big, f32x16& small) {
  small = BF16::mfma32(a.p[2], b.p[0], small);
  small = BF16::mfma32(a.p[0], b.p[2], small);
  small = BF16::mfma32(a.p[1], b.p[1], small);
  small = BF16::mfma32(a.p[1], b.p[0], small);
  small = BF16::mfma32(a.p[0], b.p[1], small);
  big = BF16::mfma32(a.p[0], b.p[0], big);
}

struct FloatRows {
  __amdgpu_buffer_rsrc_t rsrc;
  int hd;
  __device__ __forceinline__ FloatRows(const u16* base, int64_t row0, int rows, int hd_) : hd(hd_) {
    rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)((const float*)base + row0 * hd_), (short)0, rows * hd_ * 4, 0x00020000);
  }
  // 4 elements of a row: zeros past the rows and past hd, a multiple of 4
  __device__ __forceinline__ f32x4 load4(int row, int d) const {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, d < hd ? (row * hd + d) * 4 : 0x7ffffff0, 0, 0));
  }
  __device__ __forceinline__ Parts8 parts8(int row, int d) const {
    const f32x4 a = load4(row, d), b = load4(row, d + 4);
    const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return split8(v);
  }
};

// Two float tiles: memory -> registers -> three parts each in LDS, the first tile's before the second's.
template <int D>
struct PartStage {
  using P = PartTile<D>;
  static constexpr int COLS = D / 8, SLOTS = P::ROWS * COLS / THREADS;  // chunks of 8 a tile and thread
  f32x4 r[2][SLOTS][2];
  __device__ __forceinline__ void load(const FloatRows& m0, const FloatRows& m1, int row0) {
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int s = 0; s < SLOTS; s++) {
        const int id = threadIdx.x + s * THREADS, row = row0 + id / COLS, d = id % COLS * 8;
        r[w][s][0] = (w ? m1 : m0).load4(row, d);
        r[w][s][1] = (w ? m1 : m0).load4(row, d + 4);
      }
  }
  __device__ __forceinline__ void store(u16* tiles) {
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int s = 0; s < SLOTS; s++) {
        const int id = threadIdx.x + s * THREADS;
        const f32x4 a = r[w][s][0], b = r[w][s][1];
        const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        const Parts8 o = split8(v);
        u16* at = tiles + 3 * w * P::MATRIX + tile_at<D>(id / COLS, id % COLS * 8);
#pragma unroll
        for (int p = 0; p < 3; p++) *(u16x8*)(at + p * P::MATRIX) = o.p[p];
      }
  }
};

template <int D>
__device__ __forceinline__ Parts8 row_parts(const u16* tile, int r, int c) {
  Parts8 o;
#pragma unroll
  for (int p = 0; p < 3; p++) o.p[p] = read_row<D>(tile + p * PartTile<D>::MATRIX, r, c);
  return o;
}
template <int D>
__device__ __forceinline__ Parts8 transposed_parts(const u16* tile, int k0, int d0) {
  Parts8 o;
#pragma unroll
  for (int p = 0; p < 3; p++) o.p[p] = read_transposed<D>(tile + p * PartTile<D>::MATRIX, k0, d0);
  return o;
}

// the 32 streamed rows from `row` on of a tile against the resident rows
template <int D>
__device__ __forceinline__ f32x16 scores(const u16* tile, int row, const Parts8* resident, int h) {
  f32x16 big = zero16(), small = zero16();
#pragma unroll
  for (int ds = 0; ds < D / 16; ds++) six(row_parts<D>(tile, row, 2 * ds + h), resident[ds], big, small);
  return big + small;
}

// acc += (rows r0 .. r0 + 31 of the tile)^T s
template <int D>
__device__ __forceinline__ void gather(const u16* tile, int r0, const f32x16& s, f32x16* acc) {
  const Parts8 b[2] = {split_items(s, 0), split_items(s, 8)};
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++) {
    f32x16 small = zero16();
#pragma unroll
    for (int c = 0; c < 2; c++) six(transposed_parts<D>(tile, r0 + 16 * c, dt * 32), b[c], acc[dt], small);
    acc[dt] += small;
  }
}

// The streamed rows a block visits, PartTile rows at a time: the visit's tiles of 64, in halves where a tile is 32.
template <int D>
struct PartWalk {
  Visit visit;
  int tile, half;
  __device__ __forceinline__ explicit PartWalk(const Visit& v) : visit(v) {}
  __device__ __forceinline__ void start(int first) {
    visit.start(first);
    tile = visit.next();
    half = 0;
  }
  __device__ __forceinline__ bool more() const { return tile < visit.to; }
  __device__ __forceinline__ int row() const { return tile * TILE + half * 32; }
  __device__ __forceinline__ int alike() const { return D <= 64 ? visit.alike : visit.alike >> half; }
  __device__ __forceinline__ void next() {
    if (D > 64 && half == 0) {
      half = 1;
      return;
    }
    half = 0;
    tile = visit.next();
  }
};

// ---- forward ----------------------------------------------------------------------------------------------

template <int D, Cap CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, D <= 64 ? 2 : 1) void attend_fwd_parts(FastArgs g, RuleArgs ra) {
  using P = PartTile<D>;
  constexpr int R = P::ROWS;
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  __shared__ __attribute__((aligned(16))) u16 tiles[6 * P::MATRIX];
  __shared__ __attribute__((aligned(16))) int kdocs[R];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  QueryBlock qb;
  if (!query_block(g, ra, qb, wave, n)) return;
  const Rules r = rules_of(ra, qb.b);
  const int p = r.off + qb.row;
  const bool there = qb.row < r.t_q;
  qb.p = p;
  qb.doc = there ? query_doc(r, p) : -1;
  const float slope2 = head_slope<CAP, BIAS>(ra, qb.head);
  const FloatRows qrows(g.q, qb.bh * r.t_q, r.t_q, g.hd);
  const int64_t kv = (qb.b * g.kv_heads + qb.kvh) * (int64_t)r.t_k;
  const FloatRows krows(g.k, kv, r.len, g.hd), vrows(g.v, kv, r.len, g.hd);  // keys past the live ones read as zeros
  const float unit = RAW ? r.c2 : 1.f, lift = RESCALE_LOG2 / unit;

  Parts8 qf[D / 16];
  f32x16 acc[D / 32];
  float m = neg_inf(), l = 0.f;
#pragma unroll
  for (int ds = 0; ds < D / 16; ds++) qf[ds] = qrows.parts8(qb.row, ds * 16 + 8 * h);
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++) acc[dt] = zero16();

  const int4* ranges = g.ranges ? g.ranges + qb.b * g.granules : nullptr;
  PartWalk<D> walk(key_visit(g, r, qb, ranges, bits, halves[wave], wave));
  PartStage<D> st;
  const Words dwords(r.docs, r.len);
  int dnext = 0;
  walk.start(0);
  auto load = [&](int k0) __attribute__((always_inline)) {
    st.load(krows, vrows, k0);
    dnext = dwords.whole(k0 + lane);
  };
  if (walk.more()) load(walk.row());
  while (walk.more()) {
    const int k0 = walk.row(), alike = walk.alike();
    __syncthreads();  // the tile before has been read
    st.store(tiles);
    if (ranges != nullptr && threadIdx.x < R) kdocs[threadIdx.x] = dnext;
    walk.next();
    if (walk.more()) load(walk.row());
    __syncthreads();
#pragma unroll
    for (int sub = 0; sub < P::SUBS; sub++) {
      const int s0 = k0 + sub * 32;
      f32x16 s = scores<D>(tiles, sub * 32 + n, qf, h);
      const float near = (float)(p - s0 - 4 * h);
      if (CAP == CAP_EXACT) cap_scores<16>(s, r);
      if (!RAW) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float bent;
          s[i] = bend<CAP, BIAS, false>(s[i], r, slope2, near - (float)(8 * (i >> 2) + (i & 3)), bent);
        }
      }
      if (half_edge(r, qb, (alike >> sub) & 1, s0)) {
        if (ranges != nullptr) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int4 d4 = *(const int4*)&kdocs[sub * 32 + 8 * q + 4 * h];
            const int dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
            for (int e = 0; e < 4; e++) s[4 * q + e] = (qb.doc >= 0) & (dd[e] == qb.doc) ? s[4 * q + e] : neg_inf();
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = sees(r, p, s0 + 8 * (i >> 2) + 4 * h + (i & 3)) ? s[i] : neg_inf();
      }
      float mx = neg_inf();
#pragma unroll
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[i]);
      mx = pair_max(mx);
      if (__any(mx > m + lift)) {
        const float mnew = fmaxf(m, mx);
        const float alpha = mnew == neg_inf() ? 1.f : fast_exp2((m - mnew) * unit);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++) acc[dt] *= alpha;
        m = mnew;
      }
      const float base = m == neg_inf() ? 0.f : m * unit;
      float rs = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        s[i] = RAW ? fast_exp2(fmaf(s[i], unit, -base)) : fast_exp2(s[i] - base);
        rs += s[i];
      }
      l += rs;
      gather<D>(tiles + 3 * P::MATRIX, sub * 32, s, acc);
    }
  }
  const float total = pair_sum(l);
  const bool odd = any_odd(acc);
  if (threadIdx.x == 0) g.odd[qb.bh * qb.nqb + qb.q0 / ATT_ROWS] = odd;
  store_floats<D>((float*)g.o0, qb.bh * r.t_q, acc, qb.wq0, r.t_q, g.hd, total == 0.f ? 0.f : 1.f / total);
  if (h == 0 && there) g.lse[qb.bh * (int64_t)r.t_q + qb.row] = total == 0.f ? neg_inf() : m * unit * ATT_LN2 + logf(total);
}

// ---- dQ pass: also delta = rowsum(dout * out) ---------------------------------------------------------------

template <int D, Cap CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 1) void attend_dq_parts(FastArgs g, RuleArgs ra) {
  using P = PartTile<D>;
  constexpr int R = P::ROWS;
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  __shared__ __attribute__((aligned(16))) u16 tiles[6 * P::MATRIX];
  __shared__ __attribute__((aligned(16))) int kdocs[R];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  QueryBlock qb;
  if (!query_block(g, ra, qb, wave, n)) return;
  const Rules r = rules_of(ra, qb.b);
  const int p = r.off + qb.row;
  const bool there = qb.row < r.t_q;
  qb.p = p;
  qb.doc = there ? query_doc(r, p) : -1;
  const float slope2 = head_slope<CAP, BIAS>(ra, qb.head);
  const int64_t rows0 = qb.bh * r.t_q, kv = (qb.b * g.kv_heads + qb.kvh) * (int64_t)r.t_k;
  const FloatRows qrows(g.q, rows0, r.t_q, g.hd), grows(g.dout, rows0, r.t_q, g.hd), orows(g.out, rows0, r.t_q, g.hd);
  const FloatRows krows(g.k, kv, r.len, g.hd), vrows(g.v, kv, r.len, g.hd);

  Parts8 qf[D / 16], of[D / 16];
  f32x16 acc[D / 32];
  float delta = 0.f;
#pragma unroll
  for (int ds = 0; ds < D / 16; ds++) {
    qf[ds] = qrows.parts8(qb.row, ds * 16 + 8 * h);
    const f32x4 a = grows.load4(qb.row, ds * 16 + 8 * h), b = grows.load4(qb.row, ds * 16 + 8 * h + 4);
    const f32x4 x = orows.load4(qb.row, ds * 16 + 8 * h), y = orows.load4(qb.row, ds * 16 + 8 * h + 4);
    const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    of[ds] = split8(v);
#pragma unroll
    for (int e = 0; e < 4; e++) delta = fmaf(a[e], x[e], fmaf(b[e], y[e], delta));
  }
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++) acc[dt] = zero16();
  delta = pair_sum(delta);
  if (h == 0 && there) g.delta[rows0 + qb.row] = delta;
  const float l2 = there ? att_l2(g.lse_in[rows0 + qb.row]) : __builtin_inff();

  const int4* ranges = g.ranges ? g.ranges + qb.b * g.granules : nullptr;
  PartWalk<D> walk(key_visit(g, r, qb, ranges, bits, halves[wave], wave));
  PartStage<D> st;
  const Words dwords(r.docs, r.len);
  int dnext = 0;
  walk.start(0);
  auto load = [&](int k0) __attribute__((always_inline)) {
    st.load(krows, vrows, k0);
    dnext = dwords.whole(k0 + lane);
  };
  if (walk.more()) load(walk.row());
  while (walk.more()) {
    const int k0 = walk.row(), alike = walk.alike();
    __syncthreads();
    st.store(tiles);
    if (ranges != nullptr && threadIdx.x < R) kdocs[threadIdx.x] = dnext;
    walk.next();
    if (walk.more()) load(walk.row());
    __syncthreads();
#pragma unroll 1
    for (int sub = 0; sub < P::SUBS; sub++) {
      const int s0 = k0 + sub * 32;
      f32x16 s = scores<D>(tiles, sub * 32 + n, qf, h);
      const f32x16 dp = scores<D>(tiles + 3 * P::MATRIX, sub * 32 + n, of, h);
      const float near = (float)(p - s0 - 4 * h);
      if (CAP == CAP_EXACT) cap_scores<16>(s, r);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float bent = 1.f;
        const float y = bend<CAP, BIAS, true>(s[i], r, slope2, near - (float)(8 * (i >> 2) + (i & 3)), bent);
        const float e = fast_exp2(RAW ? fmaf(y, r.c2, -l2) : y - l2);
        s[i] = e * (dp[i] - delta) * (CAP != CAP_NONE ? bent : 1.f);  // times scale once, at the store
      }
      if (half_edge(r, qb, (alike >> sub) & 1, s0)) {
        if (ranges != nullptr) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int4 d4 = *(const int4*)&kdocs[sub * 32 + 8 * q + 4 * h];
            const int dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
            for (int e = 0; e < 4; e++) s[4 * q + e] = (qb.doc >= 0) & (dd[e] == qb.doc) ? s[4 * q + e] : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = sees(r, p, s0 + 8 * (i >> 2) + 4 * h + (i & 3)) ? s[i] : 0.f;
      }
      gather<D>(tiles, sub * 32, s, acc);
    }
  }
  const bool odd = any_odd(acc);
  if (threadIdx.x == 0) g.odd[qb.bh * qb.nqb + qb.q0 / ATT_ROWS] = odd;
  store_floats<D>((float*)g.o0, rows0, acc, qb.wq0, r.t_q, g.hd, g.scale);
}

// ---- dK/dV pass -------------------------------------------------------------------------------------------

template <int D, Cap CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 1) void attend_dkv_parts(FastArgs g, RuleArgs ra) {
  using P = PartTile<D>;
  constexpr int R = P::ROWS;
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  __shared__ __attribute__((aligned(16))) u16 tiles[6 * P::MATRIX];
  __shared__ __attribute__((aligned(16))) float Ls[R];
  __shared__ __attribute__((aligned(16))) float Ds[R];
  __shared__ __attribute__((aligned(16))) int qdocs[R];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const int64_t nkb = (ra.t_k + ATT_ROWS - 1) / ATT_ROWS;
  int64_t bk, blk;
  if (!att_head_and_block(g.batch * g.kv_heads, nkb, g.head_group, bk, blk)) return;
  const int64_t b = bk / g.kv_heads;
  const int kvh = (int)(bk - b * g.kv_heads), group = g.heads / g.kv_heads;
  const int k0 = (int)blk * ATT_ROWS, wk0 = k0 + wave * 32, key = wk0 + n;
  const Rules r = rules_of(ra, b);
  const int doc = r.docs != nullptr ? (key < r.len ? r.docs[key] : -1) : 0;
  const FloatRows krows(g.k, bk * r.t_k, r.len, g.hd), vrows(g.v, bk * r.t_k, r.len, g.hd);

  Parts8 kf[D / 16], vf[D / 16];
  f32x16 gk[D / 32], gv[D / 32];
#pragma unroll
  for (int ds = 0; ds < D / 16; ds++) {
    kf[ds] = krows.parts8(key, ds * 16 + 8 * h);
    vf[ds] = vrows.parts8(key, ds * 16 + 8 * h);
  }
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++) gk[dt] = gv[dt] = zero16();

  const KeyPart part(g, r, k0, group);
  const int first_q = part.first;
  Visit visit = {part.to};
  const int4* ranges = g.ranges ? g.ranges + b * g.granules : nullptr;
  if (ranges != nullptr) {
    const int first = __builtin_amdgcn_readfirstlane(doc);
    list_tiles(bits, halves[wave], ranges, g.granules, k0, __all(doc == first) ? first : -1, r.off, visit.to, wave, WAVES);
    visit.bits = bits;
    visit.half = halves[wave];
    __syncthreads();
  }

  PartStage<D> st;
  const Words dwords(r.docs, r.t_k);
  float lnext = 0.f, dnext = 0.f;
  int qnext = -1, qpos = 0;
  const int64_t base_row = (b * g.heads + kvh * (int64_t)group) * r.t_q;
  auto load = [&](int gh, int q0) __attribute__((always_inline)) {
    const int64_t rows0 = base_row + gh * (int64_t)r.t_q;
    st.load(FloatRows(g.q, rows0, r.t_q, g.hd), FloatRows(g.dout, rows0, r.t_q, g.hd), q0);
    lnext = Words(g.lse_in + rows0, r.t_q).real(q0 + lane);
    dnext = Words(g.delta + rows0, r.t_q).real(q0 + lane);
    qnext = dwords.whole(r.off + q0 + lane);
    qpos = r.off + q0 + lane;
  };
  PartWalk<D> walk(visit);
  walk.start(first_q);
  int gh = walk.more() ? part.g0 : part.g1;
  if (gh < part.g1) load(gh, walk.row());
  while (gh < part.g1) {
    const int r0 = walk.row(), alike = walk.alike();
    const float slope2 = head_slope<CAP, BIAS>(ra, kvh * group + gh);
    __syncthreads();
    st.store(tiles);
    if (threadIdx.x < R) {
      Ls[threadIdx.x] = att_l2(lnext);
      Ds[threadIdx.x] = dnext;
      qdocs[threadIdx.x] = qpos < 0 ? -1 : qnext;
    }
    walk.next();
    if (!walk.more()) {  // the next head's first
      gh++;
      walk.start(first_q);
    }
    if (gh < part.g1) load(gh, walk.row());
    __syncthreads();
#pragma unroll 1
    for (int sub = 0; sub < P::SUBS; sub++) {
      const int s0 = r0 + sub * 32;
      f32x16 s = scores<D>(tiles, sub * 32 + n, kf, h);
      f32x16 dp = scores<D>(tiles + 3 * P::MATRIX, sub * 32 + n, vf, h);
      const float near = (float)(r.off + s0 + 4 * h - key);
      if (CAP == CAP_EXACT) cap_scores<16>(s, r);
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const f32x4 l4 = *(const f32x4*)&Ls[sub * 32 + 8 * q + 4 * h], d4 = *(const f32x4*)&Ds[sub * 32 + 8 * q + 4 * h];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int i = 4 * q + e;
          float bent = 1.f;
          const float y = bend<CAP, BIAS, true>(s[i], r, slope2, near + (float)(8 * q + e), bent);
          s[i] = fast_exp2(RAW ? fmaf(y, r.c2, -l4[e]) : y - l4[e]);
          dp[i] = s[i] * (dp[i] - d4[e]) * (CAP != CAP_NONE ? bent : 1.f);  // times scale once, at the store
        }
      }
      bool edge = s0 + 32 > r.t_q || wk0 + 32 > r.len || (r.causal && r.off + s0 < wk0 + 31 && wk0 + 31 >= r.pre);
      edge |= ((alike >> sub) & 1) == 0;
      if (edge) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int4 q4 = *(const int4*)&qdocs[sub * 32 + 8 * q + 4 * h];
          const int dd[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int qq = s0 + 8 * q + 4 * h + e;
            const bool see = (qq < r.t_q) & sees(r, r.off + qq, key) & ((ranges == nullptr) | ((doc >= 0) & (dd[e] == doc)));
            s[4 * q + e] = see ? s[4 * q + e] : 0.f;
            dp[4 * q + e] = see ? dp[4 * q + e] : 0.f;
          }
        }
      }
      gather<D>(tiles + 3 * P::MATRIX, sub * 32, s, gv);
      gather<D>(tiles, sub * 32, dp, gk);
    }
  }
  const bool odd_k = any_odd(gk), odd_v = any_odd(gv);
  if (threadIdx.x == 0 && blockIdx.y == 0) g.odd[bk * nkb + blk] = g.partial == nullptr && (odd_k | odd_v);
  store_keys<D>(g, bk, r.t_k, wk0, gk, gv, g.scale, 1.f,
                [&](const f32x16* acc, u16* o, float mul) __attribute__((always_inline)) { store_floats<D>((float*)o, bk * r.t_k, acc, wk0, r.t_k, g.hd, mul); });
}

// ---- launches -----------------------------------------------------------------------------------------------

template <AttendPass PASS, int D, Cap CAP, bool BIAS>
int launch_parts_as(const FastArgs& g, const RuleArgs& ra, hipStream_t stream) {
  const int64_t blocks = PASS == ATTEND_PASS_DKV ? att_grid(g.batch * g.kv_heads, (ra.t_k + ATT_ROWS - 1) / ATT_ROWS, g.head_group)
                                                 : att_grid(g.batch * g.heads, (ra.t_q + ATT_ROWS - 1) / ATT_ROWS, g.head_group);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "attend: %lld workgroups exceed one launch", (long long)blocks);
  const dim3 grid((unsigned)blocks, PASS == ATTEND_PASS_DKV ? (unsigned)(g.head_parts * g.tile_parts) : 1), block(THREADS);
  if constexpr (PASS == ATTEND_PASS_FWD)
    hipLaunchKernelGGL((attend_fwd_parts<D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  else if constexpr (PASS == ATTEND_PASS_DQ)
    hipLaunchKernelGGL((attend_dq_parts<D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  else
    hipLaunchKernelGGL((attend_dkv_parts<D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  return check_hip(hipGetLastError(), "launching attention");
}

template <AttendPass PASS, int D>
int launch_parts_rules(const FastArgs& g, const RuleArgs& ra, hipStream_t stream) {
  const bool cap = ra.softcap > 0.f, bias = ra.slopes != nullptr;
  if (cap) return bias ? launch_parts_as<PASS, D, CAP_EXACT, true>(g, ra, stream) : launch_parts_as<PASS, D, CAP_EXACT, false>(g, ra, stream);
  return bias ? launch_parts_as<PASS, D, CAP_NONE, true>(g, ra, stream) : launch_parts_as<PASS, D, CAP_NONE, false>(g, ra, stream);
}

template <AttendPass PASS>
int launch_parts(const FastArgs& g, const RuleArgs& ra, hipStream_t stream) {
  return g.hd <= 64 ? launch_parts_rules<PASS, 64>(g, ra, stream) : launch_parts_rules<PASS, 128>(g, ra, stream);
}

}  // namespace
}  // namespace limn
