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
//    cycles and about 6 other operations of 4 an element, the cap an exponential and a reciprocal more.
//    At two waves a SIMD it is the length of that chain which counts, not its issue: the exact cap of near scores, a
//    polynomial of some 10 cycles an element less, takes no less (see Cap).
//  - the query heads of a key head are one loop of the dK/dV pass: their gradients are one sum in head order.
//
// Measured (causal, bf16; of the rate of the products it must do): 4 x 16 heads over 4 key heads x 4096 x 128, capped:
// forward 366 us (750 TFLOP/s), backward 1090 (630); 8 x 16 heads x 4096 x 128 with documents of 1024: 385 and 1080 us
// (540 and 480 TFLOP/s: of some 10 us that a workgroup takes to begin and end, 12 tiles hide less than 33);
// 32 x 8 heads x 512 x 64 with distance and documents of 200: 47 and 104 us, bound by those beginnings.
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

constexpr int ATT_WORDS = 32;     // 64-tile words of the visit list: 131072 streamed rows

// ---- which head and block a workgroup takes ----------------------------------------------------------------

// Workgroup id runs on XCD id % 8. Heads go to XCDs in groups of `group` (so that what a group's blocks stream
// stays in one L2, see head_and_block in sdpa_mfma.h), group j to XCD j % 8: where documents or lengths differ, so
// does the work of sequences, and an XCD that had all heads of one sequence (8 sequences, 8 XCDs) left the
// others waiting: packed documents, forward, 8 x 16 heads x 4096 rows: 600 us so, 444 spread. The grid is
// padded to whole groups; workgroups past the heads have nothing (false). group 0: heads in turn.
__device__ __forceinline__ bool att_head_and_block(int64_t heads, int64_t nblocks, int group, int64_t& b, int64_t& blk) {
  if (group == 0) {
    b = blockIdx.x % heads;
    blk = blockIdx.x / heads;
    return true;
  }
  const int64_t slot = blockIdx.x / 8, per = group * nblocks, j = slot / per * 8 + blockIdx.x % 8, r = slot % per;
  b = j * group + r % group;
  blk = r / group;
  return b < heads;
}

inline int64_t att_grid(int64_t heads, int64_t nblocks, int group) {
  return group == 0 ? heads * nblocks : (heads + 8 * group - 1) / (8 * group) * 8 * group * nblocks;
}

// ---- documents: ranges, visit lists ---------------------------------------------------------------------

struct DocRange {
  int lo, hi;
  __device__ __forceinline__ bool meets(const DocRange& o) const { return lo <= hi && o.lo <= o.hi && lo <= o.hi && o.lo <= hi; }
};

// A granule's entry (attend_ranges); an empty one outside [0, count). The load is unconditional: a block's loads of
// entries all go out at once, and one wait is all that a block's start has for them.
__device__ __forceinline__ int4 granule_at(const int4* granules, int count, int g) {
  const int4 e = granules[min(max(g, 0), count - 1)];
  return g < 0 || g >= count ? int4{0x7fffffff, 0, -2, 0} : e;
}

// The streamed tiles a block visits, in order from a first one on: every tile before `to`, or those with a bit
// set in LDS, 64 tiles a word. The word at hand stays in scalar registers: the next tile is a count of its
// trailing zeros, and LDS is read once in 64 tiles.
struct Visit {
  int to, at;            // at: the next tile to look at (without bits), or its word's first tile
  const uint64_t* bits;  // or nullptr
  const uint64_t* half;  // this wave's words of its halves (see alike_words): first halves, then ATT_WORDS on the second
  uint64_t word, half0, half1;
  int alike;             // of the tile that next() returned: bit 0 / 1, its first / second half has the wave's document alone
  __device__ __forceinline__ void start(int first) {
    at = first;
    alike = 3;
    if (bits != nullptr) {
      at = first & ~63;
      word = 0;
      if (at < to) {
        fetch();
        word &= ~0ull << (first & 63);
      }
    }
  }
  static __device__ __forceinline__ uint64_t scalar(uint64_t w) {
    return ((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(w >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)w);
  }
  __device__ __forceinline__ void fetch() {
    word = scalar(bits[at >> 6]);
    half0 = scalar(half[at >> 6]);
    half1 = scalar(half[ATT_WORDS + (at >> 6)]);
  }
  // the next tile, or `to` behind the last
  __device__ __forceinline__ int next() {
    if (bits == nullptr) return at < to ? at++ : to;
    while (word == 0) {
      if ((at += 64) >= to) {
        at = to;  // stays there: a word past the end is never read
        return to;
      }
      fetch();
    }
    const int bit = __builtin_ctzll(word);
    word &= word - 1;
    alike = (int)((half0 >> bit) & 1) | ((int)((half1 >> bit) & 1) << 1);
    return at + bit;
  }
};

// The lists of one block of ATT_ROWS positions from p on: bits, a bit for each streamed tile (64 positions from p0 + 64 t
// on) whose documents meet the block's, 64 tiles a word, the words shared by the waves; half, for this wave's
// document doc (-1: its rows differ), a bit for each half tile that has it alone, which then needs no test of
// documents. Entries hold granules of 32 positions: where p0 is inside one, a half tile has one document if both
// entries that it reaches into say so.
__device__ __forceinline__ void list_tiles(uint64_t* bits, uint64_t* half, const int4* granules, int count, int p, int doc, int p0, int tiles, int wave, int waves) {
  const int lane = threadIdx.x & 63;
  const bool inside = (p0 & 31) != 0;
  constexpr int OWN = ATT_ROWS / 32 + 1;
  int4 own[OWN];
#pragma unroll
  for (int j = 0; j < OWN; j++) own[j] = granule_at(granules, count, (p >> 5) + j);
  if ((p & 31) == 0) own[OWN - 1] = int4{0x7fffffff, 0, -2, 0};
  for (int w = 0; w * 64 < tiles; w++) {
    const int t = w * 64 + lane, g = (p0 >> 5) + 2 * t;
    const int4 e0 = granule_at(granules, count, g), e1 = granule_at(granules, count, g + 1), e2 = granule_at(granules, count, inside ? g + 2 : -1);
    if (w % waves == wave) {
      DocRange mine = {0x7fffffff, 0};
#pragma unroll
      for (int j = 0; j < OWN; j++) mine = {min(mine.lo, own[j].x), max(mine.hi, own[j].y)};
      const uint64_t word = __ballot(t < tiles && mine.meets(DocRange{min(min(e0.x, e1.x), e2.x), max(max(e0.y, e1.y), e2.y)}));
      if (lane == 0) bits[w] = word;
    }
    const bool in = t < tiles && doc >= 0;
    const uint64_t h0 = __ballot(in && e0.z == doc && (!inside || e1.z == doc)), h1 = __ballot(in && e1.z == doc && (!inside || e2.z == doc));
    if (lane == 0) {
      half[w] = h0;
      half[ATT_WORDS + w] = h1;
    }
  }
}

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

// Words beside a streamed tile (documents, statistics), loaded a tile ahead by every wave though one stores them: a load
// that only some waves take leaves a copy of the register to make, which waits for every load of the wave, those of the
// next tile too (backward of 8 x 16 heads x 4096 x 64 with documents of 1000: 680 us so, 659 now). A word outside
// [0, count) is 0; what it stands for is masked by its position.
struct Words {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ Words(const void* base, int count) { rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, base == nullptr ? 0 : count * 4, 0x00020000); }
  __device__ __forceinline__ int whole(int i) const { return (int)__builtin_amdgcn_raw_buffer_load_b32(rsrc, i * 4, 0, 0); }
  __device__ __forceinline__ float real(int i) const { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, i * 4, 0, 0)); }
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

// 32 rows of float results: a lane holds row n's 4 consecutive elements
template <int D>
__device__ __forceinline__ void store_floats(float* base, int64_t first, const f32x16* acc, int row0, int rows, int hd, float mul) {
  const int lane = threadIdx.x & 63, h = lane >> 5, row = row0 + (lane & 31);
  if (row >= rows) return;
  float* o = base + (first + row) * hd;
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int d = dt * 32 + 8 * q + 4 * h;
      if (d < hd) *(f32x4*)(o + d) = f32x4{acc[dt][4 * q], acc[dt][4 * q + 1], acc[dt][4 * q + 2], acc[dt][4 * q + 3]} * mul;
    }
}

// What of a key block's queries a workgroup of the dK/dV pass takes: heads [g0, g1) of the group and tiles [first, to).
struct KeyPart {
  int g0, g1, first, to;
  __device__ __forceinline__ KeyPart(const FastArgs& g, const Rules& r, int k0, int group) {
    const int y = blockIdx.y, hp = y / g.tile_parts, tp = y - hp * g.tile_parts;
    g0 = group * hp / g.head_parts;
    g1 = group * (hp + 1) / g.head_parts;
    // from the first tile that can see the block's first key on, unless a prefix opens it to all
    first = r.causal && k0 >= r.pre ? max(0, k0 - r.off) / TILE : 0;
    to = k0 < r.len ? (r.t_q + TILE - 1) / TILE : 0;
    const int tiles = max(0, to - first);
    to = min(to, first + (int)((int64_t)tiles * (tp + 1) / g.tile_parts));
    first += (int)((int64_t)tiles * tp / g.tile_parts);
  }
};

// The dK and dV totals of a key block, or of a part of it.
template <int D, typename STORE>
__device__ __forceinline__ void store_keys(const FastArgs& g, int64_t bk, int t_k, int wk0, const f32x16* gk, const f32x16* gv, float mul_k, float mul_v, STORE store) {
  if (g.partial == nullptr) {
    store(gk, g.o0, mul_k);
    store(gv, g.o1, mul_v);
    return;
  }
  const int64_t keys = g.batch * g.kv_heads * (int64_t)t_k;
  store_floats<D>(g.partial, (2 * blockIdx.y) * keys + bk * t_k, gk, wk0, t_k, g.hd, mul_k);
  store_floats<D>(g.partial, (2 * blockIdx.y + 1) * keys + bk * t_k, gv, wk0, t_k, g.hd, mul_v);
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
// passes 1), taken off again at the store. dS = p (dp - delta) goes multiplied by 2^8: an element is then off by 2^-33
// at most where it is below the normal numbers, and a sum of 2^16 such of random sign by 2^-25, which the
// result's own rounding costs it too; past 2^8 it overflows, and the block is recomputed in float. bfloat16 has
// float32's range.
template <typename T>
constexpr float shift_of(float bits) {
  return std::is_same<T, F16>::value ? bits : 0.f;
}
constexpr float DS_BITS = 8.f;
template <typename T>
constexpr float ds_down() {
  return std::is_same<T, F16>::value ? 1.f / 256.f : 1.f;
}

// ---- scores ---------------------------------------------------------------------------------------------

// How scores are capped. CAP_SHORT, half widths under caps up to CAP_SHORT_MOST: 1 - 2 / (1 + e^2z), whose error is one of the
// cap, 8 2^-24 of it, wherever z is: 2^-15 of a score at most here, a sixteenth of float16's half step on a weight.
// CAP_EXACT, everything else: cap_scores. (Forward and backward of 4 x 16 heads over 4 key heads x 4096 x 128, cap 50: 369 + 1135
// us short, 383 + 1150 exact; of 8 x 16 x 2048 x 64 161 + 459 and 177 + 454; where many scores are past half the cap
// 355 + 1106 and 513 + 1264, as the exact form computes both of its halves there.)
enum Cap { CAP_NONE, CAP_SHORT, CAP_EXACT };
constexpr float CAP_SHORT_MOST = 64.f;

// A score tile item into log2 units (as it is, if there is neither cap nor distance: then c2 comes in with
// the exponential; under CAP_EXACT cap_scores has been over the tile), and for the backward the cap's derivative.
template <Cap CAP, bool BIAS, bool GRAD>
__device__ __forceinline__ float bend(float x, const Rules& r, float slope2, float far, float& bent) {
  float y = x;
  if (CAP == CAP_EXACT) {
    if (GRAD) bent = cap_slope(r, x);
  } else if (CAP == CAP_SHORT) {
    // the derivative 1 - tanh^2 = 4 w (1 - w) with w = 1 / (1 + e^2z)
    const float w = __builtin_amdgcn_rcpf(1.f + fast_exp2(x * r.cap_in));
    y = fmaf(-2.f * r.cap_out, w, r.cap_out);
    if (GRAD) bent = 4.f * w * (1.f - w);
  } else if (BIAS) {
    y = x * r.c2;
  }
  if (BIAS) y = fmaf(-slope2, fabsf(far), y);
  return y;
}

// a head's distance penalty in log2 units
template <Cap CAP, bool BIAS>
__device__ __forceinline__ float head_slope(const RuleArgs& ra, int head) {
  if (!BIAS || (CAP == CAP_EXACT && ra.slopes == nullptr)) return 0.f;
  return ra.slopes[head] * LOG2E;
}

// ---- forward --------------------------------------------------------------------------------------------

template <typename T, int D, Cap CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 2) void attend_fwd_mfma(FastArgs g, RuleArgs ra) {
  constexpr int TE = TILE * tile_stride<D>();
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  constexpr float UP = shift_of<T>(7.f);
  __shared__ __attribute__((aligned(16))) u16 tiles[4 * TE];
  __shared__ __attribute__((aligned(16))) int kdocs[2][TILE];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const int64_t nqb = (ra.t_q + ATT_ROWS - 1) / ATT_ROWS;
  int64_t bh, blk;
  if (!att_head_and_block(g.batch * g.heads, nqb, g.head_group, bh, blk)) return;
  const int64_t b = bh / g.heads;
  const int head = (int)(bh - b * g.heads), kvh = head / (g.heads / g.kv_heads);
  const int q0 = (int)(nqb - 1 - blk) * ATT_ROWS, wq0 = q0 + wave * 32, row = wq0 + n;  // causal: the longest rows go first
  const Rules r = rules_of(ra, b);
  const int p = r.off + row;
  const bool there = row < r.t_q;
  const int doc = there ? query_doc(r, p) : -1;
  const float slope2 = head_slope<CAP, BIAS>(ra, head);
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
  Visit visit = {kend > 0 ? (kend + TILE - 1) / TILE : 0};
  const int4* ranges = g.ranges ? g.ranges + b * g.granules : nullptr;
  if (ranges != nullptr) {
    const int first = __builtin_amdgcn_readfirstlane(doc);
    list_tiles(bits, halves[wave], ranges, g.granules, r.off + q0, __all(doc == first) ? first : -1, 0, visit.to, wave, WAVES);
    visit.bits = bits;
    visit.half = halves[wave];
    __syncthreads();
  }

  HeadStage<D> st;
  int dnext = 0;
  visit.start(0);
  int cur = visit.next(), alike = visit.alike, nxt = visit.next();
  const Words dwords(r.docs, r.len);
  auto docs_load = [&](int t) { return dwords.whole(t * TILE + lane); };
  if (cur < visit.to) {
    st.load(krows, vrows, cur * TILE);
    dnext = docs_load(cur);
    st.store(tiles, tiles + TE);
    if (ranges != nullptr && wave == 0) kdocs[0][lane] = dnext;
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
      if (CAP == CAP_EXACT) cap_scores<16>(s, r);
      if (!RAW) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float unused;
          s[i] = bend<CAP, BIAS, false>(s[i], r, slope2, near - (float)(8 * (i >> 2) + (i & 3)), unused);
        }
      }
      const bool edge = s0 + 32 > r.len || (r.causal && s0 + 31 > r.off + wq0 && s0 + 31 >= r.pre);
      const bool alone = (alike >> sub) & 1;
      if (edge | !alone) {
        if (!alone) {
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
    alike = visit.alike;
    if (cur < visit.to) {
      u16* Kn = tiles + 2 * (buf ^ 1) * TE;
      st.store(Kn, Kn + TE);
      if (ranges != nullptr && wave == 0) kdocs[buf ^ 1][lane] = dnext;
      nxt = visit.next();
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

template <typename T, int D, Cap CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 2) void attend_dq_mfma(FastArgs g, RuleArgs ra) {
  constexpr int TE = TILE * tile_stride<D>();
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  __shared__ __attribute__((aligned(16))) u16 tiles[4 * TE];
  __shared__ __attribute__((aligned(16))) int kdocs[2][TILE];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const int64_t nqb = (ra.t_q + ATT_ROWS - 1) / ATT_ROWS;
  int64_t bh, blk;
  if (!att_head_and_block(g.batch * g.heads, nqb, g.head_group, bh, blk)) return;
  const int64_t b = bh / g.heads;
  const int head = (int)(bh - b * g.heads), kvh = head / (g.heads / g.kv_heads);
  const int q0 = (int)(nqb - 1 - blk) * ATT_ROWS, wq0 = q0 + wave * 32, row = wq0 + n;
  const Rules r = rules_of(ra, b);
  const int p = r.off + row;
  const bool there = row < r.t_q;
  const int doc = there ? query_doc(r, p) : -1;
  const float slope2 = head_slope<CAP, BIAS>(ra, head);
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
  const float l2 = there ? att_l2(g.lse_in[rows0 + row]) - shift_of<T>(DS_BITS) : __builtin_inff();

  const int last = min(q0 + ATT_ROWS, r.t_q) - 1;
  int kend = r.len;
  if (r.causal) kend = min(kend, max(r.off + last + 1, r.pre));
  Visit visit = {kend > 0 ? (kend + TILE - 1) / TILE : 0};
  const int4* ranges = g.ranges ? g.ranges + b * g.granules : nullptr;
  if (ranges != nullptr) {
    const int first = __builtin_amdgcn_readfirstlane(doc);
    list_tiles(bits, halves[wave], ranges, g.granules, r.off + q0, __all(doc == first) ? first : -1, 0, visit.to, wave, WAVES);
    visit.bits = bits;
    visit.half = halves[wave];
    __syncthreads();
  }

  HeadStage<D> st;
  int dnext = 0;
  visit.start(0);
  int cur = visit.next(), alike = visit.alike, nxt = visit.next();
  const Words dwords(r.docs, r.len);
  auto docs_load = [&](int t) { return dwords.whole(t * TILE + lane); };
  if (cur < visit.to) {
    st.load(krows, vrows, cur * TILE);
    dnext = docs_load(cur);
    st.store(tiles, tiles + TE);
    if (ranges != nullptr && wave == 0) kdocs[0][lane] = dnext;
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
      if (CAP == CAP_EXACT) cap_scores<16>(s, r);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float bent = 1.f;
        const float y = bend<CAP, BIAS, true>(s[i], r, slope2, near - (float)(8 * (i >> 2) + (i & 3)), bent);
        const float e = fast_exp2(RAW ? fmaf(y, r.c2, -l2) : y - l2);
        s[i] = e * (dp[i] - delta) * (CAP != CAP_NONE ? bent : 1.f);  // times scale once, at the store
      }
      const bool edge = s0 + 32 > r.len || (r.causal && s0 + 31 > r.off + wq0 && s0 + 31 >= r.pre);
      const bool alone = (alike >> sub) & 1;
      if (edge | !alone) {
        if (!alone) {
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
    alike = visit.alike;
    if (cur < visit.to) {
      u16* Kn = tiles + 2 * (buf ^ 1) * TE;
      st.store(Kn, Kn + TE);
      if (ranges != nullptr && wave == 0) kdocs[buf ^ 1][lane] = dnext;
      nxt = visit.next();
      if (nxt < visit.to) {
        st.load(krows, vrows, nxt * TILE);
        dnext = docs_load(nxt);
      }
    }
    __syncthreads();
  }
  const bool odd = any_odd(acc);
  if (threadIdx.x == 0) g.odd[bh * nqb + q0 / ATT_ROWS] = odd;
  store_rows<T, D>(g.o0 + rows0 * g.hd, acc, wq0, r.t_q, g.hd, g.scale * ds_down<T>(), tiles + wave * TE);
}

// ---- dK/dV pass up to 64 dims -----------------------------------------------------------------------------

template <typename T, int D, Cap CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 2) void attend_dkv_mfma(FastArgs g, RuleArgs ra) {
  constexpr int TE = TILE * tile_stride<D>();
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  constexpr float UP = shift_of<T>(14.f), DOWN = std::is_same<T, F16>::value ? 1.f / 16384.f : 1.f;
  constexpr float DS = DOWN / ds_down<T>();  // turns p 2^14 (dp - delta) into dS 2^8
  __shared__ __attribute__((aligned(16))) u16 tiles[4 * TE];
  __shared__ __attribute__((aligned(16))) float Ls[2][TILE];
  __shared__ __attribute__((aligned(16))) float Ds[2][TILE];
  __shared__ __attribute__((aligned(16))) int qdocs[2][TILE];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const int64_t nkb = (ra.t_k + ATT_ROWS - 1) / ATT_ROWS;
  int64_t bk, blk;
  if (!att_head_and_block(g.batch * g.kv_heads, nkb, g.head_group, bk, blk)) return;  // causal: the first keys are seen by the most queries
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

  HeadStage<D> st;
  const Words dwords(r.docs, r.t_k);
  float lnext = 0.f, dnext = 0.f;
  int qnext = -1, tnext = 0;
  const int64_t head_rows = r.t_q;
  const int64_t base_row = (b * g.heads + kvh * (int64_t)group) * head_rows;
  // tile `t` of query head `gh` of the group
  auto load = [&](int gh, int t) __attribute__((always_inline)) {
    const int64_t rows0 = base_row + gh * head_rows;
    const HeadRows qrows(g.q + rows0 * g.hd, r.t_q, g.hd), grows(g.dout + rows0 * g.hd, r.t_q, g.hd);
    st.load(qrows, grows, t * TILE);
    const int qq = t * TILE + lane;
    lnext = Words(g.lse_in + rows0, r.t_q).real(qq);
    dnext = Words(g.delta + rows0, r.t_q).real(qq);
    qnext = dwords.whole(r.off + qq);
    tnext = t;
  };
  auto store = [&](int buf) __attribute__((always_inline)) {
    u16* Qn = tiles + 2 * buf * TE;
    st.store(Qn, Qn + TE);
    if (wave == 0) {
      Ls[buf][lane] = att_l2(lnext) - UP;
      Ds[buf][lane] = dnext * DS;
      if (ranges != nullptr) qdocs[buf][lane] = r.off + tnext * TILE + lane < 0 ? -1 : qnext;
    }
  };
  visit.start(first_q);
  const int begin = visit.next();
  int gh = part.g0, cur = begin, ngh = gh, nxt = begin, alike = visit.alike;
  // the tile after (ngh, nxt): the head's next, or the next head's first
  auto advance = [&]() __attribute__((always_inline)) {
    nxt = visit.next();
    if (nxt >= visit.to) {
      ngh++;
      visit.start(first_q);
      nxt = visit.next();
    }
  };
  const bool any = begin < visit.to;
  if (any) {
    load(gh, cur);
    store(0);
    advance();
    if (ngh < part.g1) load(ngh, nxt);
  }
  __syncthreads();
  for (int buf = 0; any && gh < part.g1; buf ^= 1) {
    const int r0 = cur * TILE;
    const float slope2 = head_slope<CAP, BIAS>(ra, kvh * group + gh);
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
      if (CAP == CAP_EXACT) cap_scores<16>(s, r);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float bent = 1.f;
        const float y = bend<CAP, BIAS, true>(s[i], r, slope2, near + (float)(8 * (i >> 2) + (i & 3)), bent);
        const float l2 = l4[i >> 2][i & 3];
        s[i] = fast_exp2(RAW ? fmaf(y, r.c2, -l2) : y - l2);
        dp[i] = s[i] * fmaf(dp[i], DS, -d4[i >> 2][i & 3]) * (CAP != CAP_NONE ? bent : 1.f);  // times scale once, at the store
      }
      const bool edge = s0 + 32 > r.t_q || wk0 + 32 > r.len || (r.causal && r.off + s0 < wk0 + 31 && wk0 + 31 >= r.pre);
      const bool alone = (alike >> sub) & 1;
      if (edge | !alone) {
        if (!alone) {
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
    alike = visit.alike;
    if (gh < part.g1) {
      store(buf ^ 1);
      advance();
      if (ngh < part.g1) load(ngh, nxt);
    }
    __syncthreads();
  }
  const bool odd_k = any_odd(gk), odd_v = any_odd(gv);
  if (threadIdx.x == 0 && blockIdx.y == 0) g.odd[bk * nkb + blk] = g.partial == nullptr && (odd_k | odd_v);
  store_keys<D>(g, bk, r.t_k, wk0, gk, gv, g.scale * ds_down<T>(), DOWN,
                [&](const f32x16* acc, u16* o, float mul) __attribute__((always_inline)) { store_rows<T, D>(o + bk * (int64_t)r.t_k * g.hd, acc, wk0, r.t_k, g.hd, mul, tiles + wave * TE); });
}

// ---- dK/dV pass past 64 dims: two waves per SIMD --------------------------------------------------------------
// The 8-wave workgroup of sdpa_bwd_kv_dual (which says what each wave does, and why K and V sit in LDS): wave w
// takes keys 32 (w % 4) .. + 31 and queries 32 (w / 4) .. + 31 of every tile, tiles of 64 rows x 128 dims come by
// LDS DMA (dims past hd as zeros) into one of two buffers while the other is computed. One wave a SIMD with K
// and V in registers (as attend_dkv_mfma, 400 registers) took 1317 us where this takes 700, 850 with dS stored for the
// dQ pass (4 x 16 heads over 4 key heads, 4096 rows, capped).

// rows [row0, row0 + 64) of hd elements into a swizzled 64 x 128 tile, this wave's eighth
struct HeadDma8 {
  static constexpr int RB = 256, PASSES = TILE * RB / 1024 / KV_WAVES;
  int voff[PASSES], hd;
  __device__ __forceinline__ HeadDma8(int hd_, int wave, int lane) : hd(hd_) {
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
      const int r = (p * KV_WAVES + wave) * (1024 / RB) + lane / (RB / 16), c = (lane % (RB / 16)) ^ swz128(r);
      voff[p] = c * 8 < hd ? (r * hd + c * 8) * 2 : 0x7ffffff0;
    }
  }
  // rows past `rows` read as zeros
  __device__ __forceinline__ void copy(u16* tile, const u16* m, int row0, int rows, int wave) const {
    const int left = (rows - row0) * hd * 2;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(m + (int64_t)row0 * hd), (short)0, left > 0 ? left : 0, 0x00020000);
#pragma unroll
    for (int p = 0; p < PASSES; p++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)((char*)tile + (p * KV_WAVES + wave) * 1024), 16, voff[p], 0, 0, 0);
  }
};

constexpr int HAND_STORES = 2;  // vector stores of dS a wave and tile, see below

template <typename T, int D, Cap CAP, bool BIAS, bool HAND>
__global__ __launch_bounds__(64 * KV_WAVES, 1) void attend_dkv_wide(FastArgs g, RuleArgs ra) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  constexpr int KS = D / 16, DT = D / 32;
  constexpr float UP = shift_of<T>(14.f), DOWN = std::is_same<T, F16>::value ? 1.f / 16384.f : 1.f;
  constexpr float DS = DOWN / ds_down<T>();  // turns p 2^14 (dp - delta) into dS 2^8
  __shared__ __attribute__((aligned(1024))) u16 Q0[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 Q1[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 O0[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 O1[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 Ks[ATT_ROWS * 128];
  __shared__ __attribute__((aligned(1024))) u16 Vs[ATT_ROWS * 128];
  __shared__ __attribute__((aligned(16))) float Ls[2][TILE];
  __shared__ __attribute__((aligned(16))) float Ds[2][TILE];
  __shared__ __attribute__((aligned(16))) int qdocs[2][TILE];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[KV_WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const int kg = wave & 3, hq = wave >> 2;  // key group, query half
  const int64_t nkb = (ra.t_k + ATT_ROWS - 1) / ATT_ROWS;
  int64_t bk, blk;
  if (!att_head_and_block(g.batch * g.kv_heads, nkb, g.head_group, bk, blk)) return;
  const int64_t b = bk / g.kv_heads;
  const int kvh = (int)(bk - b * g.kv_heads), group = g.heads / g.kv_heads;
  const int k0 = (int)blk * ATT_ROWS, wk0 = k0 + kg * 32, key = wk0 + n;
  const Rules r = rules_of(ra, b);
  const bool there = key < r.len;
  const int doc = r.docs != nullptr ? (there ? r.docs[key] : -1) : 0;
  const u16* kbase = g.k + bk * (int64_t)r.t_k * g.hd;
  const u16* vbase = g.v + bk * (int64_t)r.t_k * g.hd;
  const HeadDma8 dma(g.hd, wave, lane);
  // byte offsets of this lane's LDS reads, see sdpa_bwd_kv_dual. A row's 16-deep step ds is 32 ds exclusive-or'ed
  // into its first: the K and V rows' offsets are made so as they are read, which leaves their registers free
  int rk0, rq[KS], rt[DT][2];
  {
    const SwzReads128 ad(lane);
#pragma unroll
    for (int ds = 0; ds < KS; ds++) {
      rq[ds] = ad.row[ds] + hq * 32 * 256;
    }
    rk0 = ad.row[0] + kg * 32 * 256;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int jj = 0; jj < 2; jj++) rt[dt][jj] = ad.tr[dt][jj] + hq * 32 * 256;
  }
  auto rows_at = [](const u16* base, int off) __attribute__((always_inline)) { return *(const u16x8*)((const char*)base + off); };
  auto transposed_at = [&](const u16* tile, int c, int dt) __attribute__((always_inline)) {
    const char* p = (const char*)tile + c * 16 * 256;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p + rt[dt][0]));
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p + rt[dt][1]));
    return __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x16 gk[DT], gv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++) gk[dt] = gv[dt] = zero16();

  const KeyPart part(g, r, k0, group);
  const int first_q = part.first;
  Visit visit = {part.to};
  const int4* ranges = g.ranges ? g.ranges + b * g.granules : nullptr;
  if (ranges != nullptr) {
    const int first = __builtin_amdgcn_readfirstlane(doc);
    list_tiles(bits, halves[wave], ranges, g.granules, k0, __all(doc == first) ? first : -1, r.off, visit.to, wave, KV_WAVES);
    visit.bits = bits;
    visit.half = halves[wave];
    __syncthreads();
  }

  const int64_t base_row = (b * g.heads + kvh * (int64_t)group) * r.t_q;
  // tile `t` of query head `gh` of the group: its rows by DMA, its statistics through registers (the first wave)
  // and its documents (the second), stored only when the tile before it is done: loads retire in order
  const Words dwords(r.docs, r.t_k);
  float lnext = 0.f, dnext = 0.f;
  int qnext = -1, tnext = 0;
  auto load = [&](int gh, int t, u16* Q, u16* O) __attribute__((always_inline)) {
    const int64_t rows0 = base_row + (int64_t)gh * r.t_q;
    dma.copy(Q, g.q + rows0 * g.hd, t * TILE, r.t_q, wave);
    dma.copy(O, g.dout + rows0 * g.hd, t * TILE, r.t_q, wave);
    const int qq = t * TILE + lane;
    lnext = Words(g.lse_in + rows0, r.t_q).real(qq);
    dnext = Words(g.delta + rows0, r.t_q).real(qq);
    qnext = dwords.whole(r.off + qq);
    tnext = t;
  };
  auto stats_store = [&](int buf) __attribute__((always_inline)) {
    if (wave == 0) {
      Ls[buf][lane] = att_l2(lnext) - UP;
      Ds[buf][lane] = dnext * DS;
    }
    if (wave == 1 && ranges != nullptr) qdocs[buf][lane] = r.off + tnext * TILE + lane < 0 ? -1 : qnext;
  };

  visit.start(first_q);
  const int begin = visit.next();
  int gh = part.g0, cur = begin, ngh = gh, nxt = begin, alike = visit.alike;
  auto advance = [&]() __attribute__((always_inline)) {
    nxt = visit.next();
    if (nxt >= visit.to) {
      ngh++;
      visit.start(first_q);
      nxt = visit.next();
    }
  };

  // this wave's 32 queries of the tile against its 32 keys
  auto tile = [&](int buf, const u16* Qc, const u16* Oc) __attribute__((always_inline)) {
    const int s0 = cur * TILE + hq * 32;
    const float slope2 = head_slope<CAP, BIAS>(ra, kvh * group + gh);
    int rk = rk0;
    asm volatile("" : "+v"(rk)::"memory");  // keeps the K and V reads and their offsets in the loop: hoisted, they would fill the registers
    f32x16 s = zero16(), dp = zero16();
    u16x8 xa[2][4];
    auto xread = [&](int ds, u16x8* o) __attribute__((always_inline)) {
      const int rkd = rk ^ (32 * ds);
      o[0] = rows_at(Qc, rq[ds]); o[1] = rows_at(Ks, rkd); o[2] = rows_at(Oc, rq[ds]); o[3] = rows_at(Vs, rkd);
    };
    xread(0, xa[0]);
#pragma unroll
    for (int ds = 0; ds < KS; ds++) {
      if (ds + 1 < KS) xread(ds + 1, xa[(ds + 1) & 1]);
      s = T::mfma32(xa[ds & 1][0], xa[ds & 1][1], s);
      dp = T::mfma32(xa[ds & 1][2], xa[ds & 1][3], dp);
      __builtin_amdgcn_sched_barrier(0);
    }
    bool edge = s0 + 32 > r.t_q || wk0 + 32 > r.len || (r.causal && r.off + s0 < wk0 + 31 && wk0 + 31 >= r.pre);
    edge |= ((alike >> hq) & 1) == 0;
    const float near = (float)(r.off + s0 + 4 * h - key);
    if (CAP == CAP_EXACT) cap_scores<16>(s, r);
    // the scores straight into packed operands, in two instances: with element tests and without
    unsigned pk[8], gp[8];
    auto soft = [&](auto tests) __attribute__((always_inline)) {
      f32x4 l4, d4;
      int4 q4 = {0, 0, 0, 0};
      float pv = 0.f, gv2 = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        if ((i & 3) == 0) {
          l4 = *(const f32x4*)&Ls[buf][hq * 32 + 8 * (i >> 2) + 4 * h];
          d4 = *(const f32x4*)&Ds[buf][hq * 32 + 8 * (i >> 2) + 4 * h];
          if (decltype(tests)::value && ranges != nullptr) q4 = *(const int4*)&qdocs[buf][hq * 32 + 8 * (i >> 2) + 4 * h];
        }
        float bent = 1.f;
        const float y = bend<CAP, BIAS, true>(s[i], r, slope2, near + (float)(8 * (i >> 2) + (i & 3)), bent);
        float e = fast_exp2(RAW ? fmaf(y, r.c2, -l4[i & 3]) : y - l4[i & 3]);
        float d = e * fmaf(dp[i], DS, -d4[i & 3]) * (CAP != CAP_NONE ? bent : 1.f);  // times scale once, at the store
        if (decltype(tests)::value) {
          const int qq = s0 + 8 * (i >> 2) + 4 * h + (i & 3), qd = (i & 3) == 0 ? q4.x : (i & 3) == 1 ? q4.y : (i & 3) == 2 ? q4.z : q4.w;
          const bool see = (qq < r.t_q) & (doc >= 0) & (qd == doc) & sees(r, r.off + qq, key);
          e = see ? e : 0.f;
          d = see ? d : 0.f;
        }
        if (i & 1) {
          pk[i >> 1] = T::pack2(pv, e);
          gp[i >> 1] = T::pack2(gv2, d);
        } else {
          pv = e;
          gv2 = d;
        }
      }
    };
    if (edge)
      soft(std::true_type{});
    else
      soft(std::false_type{});
    if (HAND) {
      // the wave's 32 keys x 32 queries for attend_dq_handed: the halves of a wave trade, so that a lane stores 8 queries
      // of its key, even eights the first half and odd ones the second, 1 KB a store
      const int64_t at = ((b * g.heads + kvh * (int64_t)group + gh) * g.row_blocks + (cur >> 1)) * g.key_tiles + blk * 2 + (kg >> 1);
      u16* o = g.ds + at * (TILE * ATT_ROWS) + (((cur & 1) * 2 + hq) * 4 + (kg & 1) * 2) * 512 + lane * 8;
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const auto x = __builtin_amdgcn_permlane32_swap(gp[4 * q], gp[4 * q + 2], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(gp[4 * q + 1], gp[4 * q + 3], false, false);
        *(u32x4*)(o + 512 * q) = u32x4{x[0], y[0], x[1], y[1]};
      }
    }
    u16x8 pb[2], gb[2];
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const u32x4 wp = {pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]}, wg = {gp[4 * c], gp[4 * c + 1], gp[4 * c + 2], gp[4 * c + 3]};
      pb[c] = __builtin_bit_cast(u16x8, wp);
      gb[c] = __builtin_bit_cast(u16x8, wg);
    }
    u16x8 ya[2][2];
    auto yread = [&](int j, u16x8* o) __attribute__((always_inline)) {
      o[0] = transposed_at(Oc, j / DT, j % DT); o[1] = transposed_at(Qc, j / DT, j % DT);
    };
    yread(0, ya[0]);
#pragma unroll
    for (int j = 0; j < 2 * DT; j++) {
      if (j + 1 < 2 * DT) yread(j + 1, ya[(j + 1) & 1]);
      gv[j % DT] = T::mfma32(ya[j & 1][0], pb[j / DT], gv[j % DT]);
      gk[j % DT] = T::mfma32(ya[j & 1][1], gb[j / DT], gk[j % DT]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // one tile while the next is copied; behind the last one the last head's is copied again, for nothing
  auto step = [&](int buf, const u16* Qc, const u16* Oc, u16* Qn, u16* On) __attribute__((always_inline)) {
    load(min(ngh, part.g1 - 1), nxt, Qn, On);
    __builtin_amdgcn_sched_barrier(0);
    tile(buf, Qc, Oc);
    __builtin_amdgcn_s_waitcnt(HAND ? WAIT_VMEM + HAND_STORES : WAIT_VMEM);  // the tile's stores, issued behind the copies, stay under way
    stats_store(buf ^ 1);
    __syncthreads();
    gh = ngh;
    cur = nxt;
    alike = visit.alike;
    advance();
  };
  if (begin < visit.to) {
    int total = visit.to - begin;  // tiles of a head
    if (ranges != nullptr) {
      total = 0;
      for (int w = begin >> 6; w * 64 < visit.to; w++) {
        const uint64_t word = bits[w];
        total += __builtin_popcountll(w == begin >> 6 ? word & (~0ull << (begin & 63)) : word);
      }
      total = __builtin_amdgcn_readfirstlane(total);
    }
    total *= part.g1 - part.g0;
    dma.copy(Ks, kbase, k0, r.len, wave);
    dma.copy(Ks + TILE * 128, kbase, k0 + TILE, r.len, wave);
    dma.copy(Vs, vbase, k0, r.len, wave);
    dma.copy(Vs + TILE * 128, vbase, k0 + TILE, r.len, wave);
    load(gh, begin, Q0, O0);
    __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
    stats_store(0);
    __syncthreads();
    advance();
    int t = 0;
    for (; t + 1 < total; t += 2) {
      step(0, Q0, O0, Q1, O1);
      step(1, Q1, O1, Q0, O0);
    }
    if (t < total) step(0, Q0, O0, Q1, O1);
  }
  __syncthreads();  // every wave is done with every buffer
  const bool odd_k = any_odd(gk), odd_v = any_odd(gv);
  if (threadIdx.x == 0 && blockIdx.y == 0) g.odd[bk * nkb + blk] = g.partial == nullptr && (odd_k | odd_v);
  // the second query half's partial sums to LDS, added to the first's: always in that order
  char* const part_k = kg == 0 ? (char*)Ks : kg == 1 ? (char*)Vs : kg == 2 ? (char*)Q0 : (char*)O0;
  char* const part_v = kg == 0 ? (char*)Ks + 16384 : kg == 1 ? (char*)Vs + 16384 : kg == 2 ? (char*)Q1 : (char*)O1;
  if (hq == 1) {
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        *(f32x4*)(part_k + ((dt * 4 + e) * 64 + lane) * 16) = f32x4{gk[dt][4 * e], gk[dt][4 * e + 1], gk[dt][4 * e + 2], gk[dt][4 * e + 3]};
        *(f32x4*)(part_v + ((dt * 4 + e) * 64 + lane) * 16) = f32x4{gv[dt][4 * e], gv[dt][4 * e + 1], gv[dt][4 * e + 2], gv[dt][4 * e + 3]};
      }
  }
  __syncthreads();
  if (hq == 0) {
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const f32x4 pk4 = *(const f32x4*)(part_k + ((dt * 4 + e) * 64 + lane) * 16);
        const f32x4 pv4 = *(const f32x4*)(part_v + ((dt * 4 + e) * 64 + lane) * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          gk[dt][4 * e + j] += pk4[j];
          gv[dt][4 * e + j] += pv4[j];
        }
      }
    u16* stage = (u16*)part_k;  // which only this wave reads from now on
    store_keys<D>(g, bk, r.t_k, wk0, gk, gv, g.scale * ds_down<T>(), DOWN,
                  [&](const f32x16* acc, u16* o, float mul) __attribute__((always_inline)) { store_rows<T, D>(o + bk * (int64_t)r.t_k * g.hd, acc, wk0, r.t_k, g.hd, mul, stage); });
  }
#endif
}

// ---- forward and dQ pass past 64 dims: tiles by LDS DMA ---------------------------------------------------------
// As attend_fwd_mfma and attend_dq_mfma, with the streamed tiles copied straight into swizzled LDS tiles of 64 x 128
// (dims past hd as zeros), and the forward pipelined as sdpa_fwd_dma is: a tile's exponentials and its V product
// are issued beside the next tile's scores. Staged through registers the forward took 753 us and the dQ pass 881,
// so 577 and 773 (8 x 16 heads x 4096 rows, causal).

// rows [row0, row0 + 64) of hd elements into a swizzled 64 x 128 tile, this wave's quarter
struct HeadDma4 {
  static constexpr int RB = 256, PASSES = TILE * RB / 1024 / WAVES;
  int voff[PASSES], hd;
  __device__ __forceinline__ HeadDma4(int hd_, int wave, int lane) : hd(hd_) {
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
      const int r = (p * WAVES + wave) * (1024 / RB) + lane / (RB / 16), c = (lane % (RB / 16)) ^ swz128(r);
      voff[p] = c * 8 < hd ? (r * hd + c * 8) * 2 : 0x7ffffff0;
    }
  }
  // rows past `rows` read as zeros
  __device__ __forceinline__ void copy(u16* tile, const u16* m, int row0, int rows, int wave) const {
    const int left = (rows - row0) * hd * 2;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(m + (int64_t)row0 * hd), (short)0, left > 0 ? left : 0, 0x00020000);
#pragma unroll
    for (int p = 0; p < PASSES; p++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)((char*)tile + (p * WAVES + wave) * 1024), 16, voff[p], 0, 0, 0);
  }
};

// What a block of 128 query rows of one head is, for both passes.
struct QueryBlock {
  int64_t b, bh, nqb;
  int head, kvh, q0, wq0, row, p, doc;
};

// The key tiles such a block visits: lists in LDS where there are documents.
__device__ __forceinline__ Visit key_visit(const FastArgs& g, const Rules& r, const QueryBlock& qb, const int4* ranges, uint64_t* bits, uint64_t* half, int wave) {
  const int last = min(qb.q0 + ATT_ROWS, r.t_q) - 1;
  int kend = r.len;
  if (r.causal) kend = min(kend, max(r.off + last + 1, r.pre));
  Visit visit = {kend > 0 ? (kend + TILE - 1) / TILE : 0};
  if (ranges != nullptr) {
    const int first = __builtin_amdgcn_readfirstlane(qb.doc);
    list_tiles(bits, half, ranges, g.granules, r.off + qb.q0, __all(qb.doc == first) ? first : -1, 0, visit.to, wave, WAVES);
    visit.bits = bits;
    visit.half = half;
    __syncthreads();
  }
  return visit;
}

// tiles of a visit that starts at 0
__device__ __forceinline__ int visit_count(const Visit& v) {
  if (v.bits == nullptr) return v.to;
  int n = 0;
  for (int w = 0; w * 64 < v.to; w++) n += __builtin_popcountll(v.bits[w]);
  return __builtin_amdgcn_readfirstlane(n);
}

__device__ __forceinline__ bool query_block(const FastArgs& g, const RuleArgs& ra, QueryBlock& qb, int wave, int n) {
  qb.nqb = (ra.t_q + ATT_ROWS - 1) / ATT_ROWS;
  int64_t blk;
  if (!att_head_and_block(g.batch * g.heads, qb.nqb, g.head_group, qb.bh, blk)) return false;
  qb.b = qb.bh / g.heads;
  qb.head = (int)(qb.bh - qb.b * g.heads);
  qb.kvh = qb.head / (g.heads / g.kv_heads);
  qb.q0 = (int)(qb.nqb - 1 - blk) * ATT_ROWS;  // causal: the longest rows go first
  qb.wq0 = qb.q0 + wave * 32;
  qb.row = qb.wq0 + n;
  return true;
}

// Whether a half tile of 32 keys needs element tests for the wave's rows; alike: its bit of Visit::alike.
__device__ __forceinline__ bool half_edge(const Rules& r, const QueryBlock& qb, int alike, int s0) {
  return alike == 0 || s0 + 32 > r.len || (r.causal && s0 + 31 > r.off + qb.wq0 && s0 + 31 >= r.pre);
}

template <typename T, int D, Cap CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 2) void attend_fwd_wide(FastArgs g, RuleArgs ra) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  constexpr int KS = D / 16, DT = D / 32;
  constexpr float UP = shift_of<T>(7.f);
  __shared__ __attribute__((aligned(1024))) u16 K0[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 K1[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 V0[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 V1[TILE * 128];
  __shared__ __attribute__((aligned(16))) int kdocs[2][TILE];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  QueryBlock qb;
  if (!query_block(g, ra, qb, wave, n)) return;
  const Rules r = rules_of(ra, qb.b);
  const bool there = qb.row < r.t_q;
  const HeadRows qrows(g.q + qb.bh * (int64_t)r.t_q * g.hd, r.t_q, g.hd);
  u16x8 qf[KS];
#pragma unroll
  for (int ds = 0; ds < KS; ds++) qf[ds] = qrows.load8(qb.row, ds * 16 + 8 * h);
  qb.p = r.off + qb.row;
  qb.doc = there ? query_doc(r, qb.p) : -1;
  const int4* ranges = g.ranges ? g.ranges + qb.b * g.granules : nullptr;
  const bool docs = ranges != nullptr;
  const float slope2 = head_slope<CAP, BIAS>(ra, qb.head);
  const int64_t kv = (qb.b * g.kv_heads + qb.kvh) * (int64_t)r.t_k * g.hd;
  const u16* kbase = g.k + kv;
  const u16* vbase = g.v + kv;
  const HeadDma4 dma(g.hd, wave, lane);
  const SwzReads128 ad(lane);
  const float unit = RAW ? r.c2 : 1.f, lift = RESCALE_LOG2 / unit;

  f32x16 acc[DT], s[2];
  float m = neg_inf(), l = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; dt++) acc[dt] = zero16();

  Visit visit = key_visit(g, r, qb, ranges, bits, halves[wave], wave);
  const int count = visit_count(visit);
  visit.start(0);
  int dnext = -1;
  const Words dwords(r.docs, r.len);
  auto docs_load = [&](int t) __attribute__((always_inline)) {
    dnext = dwords.whole(t * TILE + lane);
  };
  auto docs_store = [&](int buf) __attribute__((always_inline)) {
    if (docs && wave == 0) kdocs[buf][lane] = dnext;
  };
  auto scores = [&](const u16* Kt, f32x16 (&o)[2]) __attribute__((always_inline)) {
    o[0] = zero16();
    o[1] = zero16();
#pragma unroll
    for (int ds = 0; ds < KS; ds++)
#pragma unroll
      for (int sub = 0; sub < 2; sub++) o[sub] = T::mfma32(ad.rows(Kt, sub, ds), qf[ds], o[sub]);
  };
  // a tile's scores bent and masked, and the reference point moved where they pass it by more than 2^8
  auto look = [&](f32x16 (&o)[2], int t, int buf, int alike) __attribute__((always_inline)) {
    const float near = (float)(qb.p - t * TILE - 4 * h);
#pragma unroll
    for (int sub = 0; sub < 2; sub++) {
      const int s0 = t * TILE + sub * 32;
      if (CAP == CAP_EXACT) cap_scores<16>(o[sub], r);
      if (!RAW) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float unused;
          o[sub][i] = bend<CAP, BIAS, false>(o[sub][i], r, slope2, near - (float)(sub * 32 + 8 * (i >> 2) + (i & 3)), unused);
        }
      }
      if (half_edge(r, qb, (alike >> sub) & 1, s0)) {
        if (docs && !((alike >> sub) & 1)) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int4 d4 = *(const int4*)&kdocs[buf][sub * 32 + 8 * q + 4 * h];
            const int dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
            for (int e = 0; e < 4; e++) o[sub][4 * q + e] = (qb.doc >= 0) & (dd[e] == qb.doc) ? o[sub][4 * q + e] : neg_inf();
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) o[sub][i] = sees(r, qb.p, s0 + 8 * (i >> 2) + 4 * h + (i & 3)) ? o[sub][i] : neg_inf();
      }
    }
    float mx = neg_inf();
#pragma unroll
    for (int sub = 0; sub < 2; sub++)
#pragma unroll
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, o[sub][i]);
    mx = pair_max(mx);
    if (__any(mx > m + lift)) {
      const float mnew = fmaxf(m, mx);
      const float alpha = mnew == neg_inf() ? 1.f : fast_exp2((m - mnew) * unit);
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; dt++) acc[dt] *= alpha;
      m = mnew;
    }
  };
  // a tile's probabilities (its scores in s) and V product, beside the next tile's scores
  auto pipe = [&](auto has_next, const u16* Kn, const u16* Vc, int tn, int bufn, int alike) __attribute__((always_inline)) {
    f32x16 sn[2];
    if (decltype(has_next)::value) scores(Kn, sn);
    const float base = (m == neg_inf() ? 0.f : m * unit) - UP;
    float rs = 0.f;
#pragma unroll
    for (int sub = 0; sub < 2; sub++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float e = RAW ? fast_exp2(fmaf(s[sub][i], unit, -base)) : fast_exp2(s[sub][i] - base);
        s[sub][i] = e;
        rs += e;
      }
    l += rs;
#pragma unroll
    for (int sub = 0; sub < 2; sub++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const u16x8 pb = pack8<T>(s[sub], 8 * c);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) acc[dt] = T::mfma32(ad.transposed(Vc, sub * 32 + 16 * c, dt), pb, acc[dt]);
      }
    if (decltype(has_next)::value) {
      look(sn, tn, bufn, alike);
      s[0] = sn[0];
      s[1] = sn[1];
    }
  };
  if (count > 0) {
    // tile it's K is in buffer it % 2 and its documents too, its V in buffer it % 2; K goes two tiles ahead, V one
    const int t0 = visit.next(), alike0 = visit.alike;
    int t1 = visit.next(), alike1 = visit.alike, t2 = visit.next();
    dma.copy(K0, kbase, t0 * TILE, r.len, wave);
    dma.copy(V0, vbase, t0 * TILE, r.len, wave);
    dma.copy(K1, kbase, t1 * TILE, r.len, wave);
    docs_load(t0);
    docs_store(0);
    docs_load(t1);
    __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
    docs_store(1);
    __syncthreads();
    scores(K0, s);
    look(s, t0, 0, alike0);
    __syncthreads();  // every wave's reads of K buffer 0 are done before the third tile is copied there
    // step: probabilities and V product of the tile in buffer `cur`, scores of the next
    auto step = [&](int nextbuf, const u16* Kn, const u16* Vc, u16* Kf, u16* Vf) __attribute__((always_inline)) {
      dma.copy(Kf, kbase, t2 * TILE, r.len, wave);
      dma.copy(Vf, vbase, t1 * TILE, r.len, wave);
      docs_load(t2);
      pipe(std::true_type{}, Kn, Vc, t1, nextbuf, alike1);
      __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
      docs_store(nextbuf ^ 1);
      __syncthreads();
      t1 = t2;
      alike1 = visit.alike;
      t2 = visit.next();
    };
    int it = 0;
    for (; it + 2 < count; it += 2) {
      step(1, K1, V0, K0, V1);
      step(0, K0, V1, K1, V0);
    }
    if (it + 1 < count) {
      step(1, K1, V0, K0, V1);
      pipe(std::false_type{}, K0, V1, 0, 0, 0);
    } else {
      pipe(std::false_type{}, K0, V0, 0, 0, 0);
    }
  }
  const float total = pair_sum(l);
  const bool odd = any_odd(acc);  // a barrier: the tile buffers become staging below
  if (threadIdx.x == 0) g.odd[qb.bh * qb.nqb + qb.q0 / ATT_ROWS] = odd;
  const float inv = total == 0.f ? 0.f : 1.f / total;  // a row that sees nothing is a row of zeros
  u16* stage = wave == 0 ? K0 : wave == 1 ? K1 : wave == 2 ? V0 : V1;
  store_rows<T, D>(g.o0 + qb.bh * (int64_t)r.t_q * g.hd, acc, qb.wq0, r.t_q, g.hd, inv, stage);
  if (h == 0 && there) g.lse[qb.bh * (int64_t)r.t_q + qb.row] = total == 0.f ? neg_inf() : (m * unit - UP) * ATT_LN2 + logf(total);
#endif
}

template <typename T, int D, Cap CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 2) void attend_dq_wide(FastArgs g, RuleArgs ra) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  constexpr int KS = D / 16, DT = D / 32;
  __shared__ __attribute__((aligned(1024))) u16 K0[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 K1[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 V0[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 V1[TILE * 128];
  __shared__ __attribute__((aligned(16))) int kdocs[2][TILE];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  QueryBlock qb;
  if (!query_block(g, ra, qb, wave, n)) return;
  const Rules r = rules_of(ra, qb.b);
  const bool there = qb.row < r.t_q;
  const int64_t rows0 = qb.bh * (int64_t)r.t_q;
  const HeadRows qrows(g.q + rows0 * g.hd, r.t_q, g.hd), grows(g.dout + rows0 * g.hd, r.t_q, g.hd), orows(g.out + rows0 * g.hd, r.t_q, g.hd);
  u16x8 qf[KS], of[KS];
  float delta = 0.f;
#pragma unroll
  for (int ds = 0; ds < KS; ds++) {
    qf[ds] = qrows.load8(qb.row, ds * 16 + 8 * h);
    of[ds] = grows.load8(qb.row, ds * 16 + 8 * h);
    const u16x8 o = orows.load8(qb.row, ds * 16 + 8 * h);
#pragma unroll
    for (int e = 0; e < 8; e++) delta = fmaf(T::unpack(of[ds][e]), T::unpack(o[e]), delta);
  }
  delta = pair_sum(delta);
  if (h == 0 && there) g.delta[rows0 + qb.row] = delta;
  const float l2 = there ? att_l2(g.lse_in[rows0 + qb.row]) - shift_of<T>(DS_BITS) : __builtin_inff();
  qb.p = r.off + qb.row;
  qb.doc = there ? query_doc(r, qb.p) : -1;
  const int4* ranges = g.ranges ? g.ranges + qb.b * g.granules : nullptr;
  const bool docs = ranges != nullptr;
  const float slope2 = head_slope<CAP, BIAS>(ra, qb.head);
  const int64_t kv = (qb.b * g.kv_heads + qb.kvh) * (int64_t)r.t_k * g.hd;
  const u16* kbase = g.k + kv;
  const u16* vbase = g.v + kv;
  const HeadDma4 dma(g.hd, wave, lane);
  const SwzReads128 ad(lane);

  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++) acc[dt] = zero16();

  Visit visit = key_visit(g, r, qb, ranges, bits, halves[wave], wave);
  const int count = visit_count(visit);
  visit.start(0);
  int dnext = -1;
  const Words dwords(r.docs, r.len);
  auto docs_load = [&](int t) __attribute__((always_inline)) {
    dnext = dwords.whole(t * TILE + lane);
  };
  auto docs_store = [&](int buf) __attribute__((always_inline)) {
    if (docs && wave == 0) kdocs[buf][lane] = dnext;
  };
  int cur = visit.next(), alike = visit.alike, nxt = visit.next();
  auto tile = [&](int buf, const u16* Kt, const u16* Vt) __attribute__((always_inline)) {
#pragma unroll
    for (int sub = 0; sub < 2; sub++) {
      const int s0 = cur * TILE + sub * 32;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ds = 0; ds < KS; ds++) {
        s = T::mfma32(ad.rows(Kt, sub, ds), qf[ds], s);
        dp = T::mfma32(ad.rows(Vt, sub, ds), of[ds], dp);
      }
      const float near = (float)(qb.p - s0 - 4 * h);
      if (CAP == CAP_EXACT) cap_scores<16>(s, r);
      unsigned gp[8];  // packed operands, in two instances: with element tests and without
      auto soft = [&](auto tests) __attribute__((always_inline)) {
        int4 d4 = {0, 0, 0, 0};
        float first = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
          if (decltype(tests)::value && docs && (i & 3) == 0) d4 = *(const int4*)&kdocs[buf][sub * 32 + 8 * (i >> 2) + 4 * h];
          float bent = 1.f;
          const float y = bend<CAP, BIAS, true>(s[i], r, slope2, near - (float)(8 * (i >> 2) + (i & 3)), bent);
          const float e = fast_exp2(RAW ? fmaf(y, r.c2, -l2) : y - l2);
          float d = e * (dp[i] - delta) * (CAP != CAP_NONE ? bent : 1.f);  // times scale once, at the store
          if (decltype(tests)::value) {
            const int kd = (i & 3) == 0 ? d4.x : (i & 3) == 1 ? d4.y : (i & 3) == 2 ? d4.z : d4.w;
            d = (qb.doc >= 0) & (kd == qb.doc) & sees(r, qb.p, s0 + 8 * (i >> 2) + 4 * h + (i & 3)) ? d : 0.f;
          }
          if (i & 1)
            gp[i >> 1] = T::pack2(first, d);
          else
            first = d;
        }
      };
      if (half_edge(r, qb, (alike >> sub) & 1, s0))
        soft(std::true_type{});
      else
        soft(std::false_type{});
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const u32x4 w = {gp[4 * c], gp[4 * c + 1], gp[4 * c + 2], gp[4 * c + 3]};
        const u16x8 gb = __builtin_bit_cast(u16x8, w);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) acc[dt] = T::mfma32(ad.transposed(Kt, sub * 32 + 16 * c, dt), gb, acc[dt]);
      }
    }
  };
  auto step = [&](int buf, const u16* Kc, const u16* Vc, u16* Kn, u16* Vn) __attribute__((always_inline)) {
    dma.copy(Kn, kbase, nxt * TILE, r.len, wave);
    dma.copy(Vn, vbase, nxt * TILE, r.len, wave);
    docs_load(nxt);
    tile(buf, Kc, Vc);
    __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
    docs_store(buf ^ 1);
    __syncthreads();
    cur = nxt;
    alike = visit.alike;
    nxt = visit.next();
  };
  if (count > 0) {
    dma.copy(K0, kbase, cur * TILE, r.len, wave);
    dma.copy(V0, vbase, cur * TILE, r.len, wave);
    docs_load(cur);
    __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
    docs_store(0);
    __syncthreads();
    int it = 0;
    for (; it + 1 < count; it += 2) {
      step(0, K0, V0, K1, V1);
      step(1, K1, V1, K0, V0);
    }
    if (it < count) step(0, K0, V0, K1, V1);
  }
  const bool odd = any_odd(acc);  // a barrier: the tile buffers become staging below
  if (threadIdx.x == 0) g.odd[qb.bh * qb.nqb + qb.q0 / ATT_ROWS] = odd;
  u16* stage = wave == 0 ? K0 : wave == 1 ? K1 : wave == 2 ? V0 : V1;
  store_rows<T, D>(g.o0 + rows0 * g.hd, acc, qb.wq0, r.t_q, g.hd, g.scale * ds_down<T>(), stage);
#endif
}

// ---- dQ pass past 64 dims from the dS that the dK/dV pass left ------------------------------------------------------
// dS comes in matrices of 64 keys x 128 queries (16 KB; a head's query blocks by its key tiles): 4 KB for every 32 queries,
// a wave's, of 1 KB for 32 keys and every second 16 bytes of theirs, each in the order in which a wave of the dK/dV pass
// stores it (chunks of 8 queries: of the first eight of 16, key by key, then of the second). A wave copies its own 4 KB
// into LDS, chunks of a KB exchanged so that the four 64-byte pieces which a half wave reads transposed lie in
// different banks. One product where attend_dq_wide has three, bound by the reads of dS (1.1 GB in 278 us, 4 TB/s, at 4 x 16 heads x 4096). The dK/dV pass wrote those
// matrices' halves of 64 queries that its own lists and causality name; the others are not read.

template <typename T, int D>
__global__ __launch_bounds__(THREADS, 2) void attend_dq_handed(FastArgs g, RuleArgs ra) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr int DT = D / 32;
  __shared__ __attribute__((aligned(1024))) u16 K0[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 K1[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 S0[TILE * 128];
  __shared__ __attribute__((aligned(1024))) u16 S1[TILE * 128];
  __shared__ uint64_t bits[ATT_WORDS];
  __shared__ uint64_t halves[WAVES][2 * ATT_WORDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31;
  QueryBlock qb;
  if (!query_block(g, ra, qb, wave, n)) return;
  const Rules r = rules_of(ra, qb.b);
  const u16* kbase = g.k + (qb.b * g.kv_heads + qb.kvh) * (int64_t)r.t_k * g.hd;
  const u16* sbase = g.ds + (qb.bh * g.row_blocks + qb.q0 / ATT_ROWS) * g.key_tiles * (int64_t)(TILE * ATT_ROWS);
  const HeadDma4 dma(g.hd, wave, lane);
  const SwzReads128 ad(lane);
  int rs[2], sv[2];  // byte offsets of the transposing reads of dS, and of its copy's chunks by the parity of the KB
#pragma unroll
  for (int jj = 0; jj < 2; jj++) {
    const int i = lane & 15, q = (lane >> 4) & 1, e = (i >> 1) & 1, key = 4 * (lane >> 5) + 8 * jj + (i >> 2);
    rs[jj] = wave * 4096 + q * 1024 + (e * 32 + (key ^ (4 * (e + 2 * q)))) * 16 + (i & 1) * 8;
    sv[jj] = (lane ^ (4 * ((lane >> 5) + 2 * jj))) * 16;
  }
  auto columns = [&](const u16* tile, int c) __attribute__((always_inline)) {  // keys 16 c .. + 15
    const char* p = (const char*)tile + (c >> 1) * 2048 + (c & 1) * 256;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p + rs[0]));
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p + rs[1]));
    return __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++) acc[dt] = zero16();

  const int last = min(qb.q0 + ATT_ROWS, r.t_q) - 1, tile = qb.wq0 / TILE;  // tile: the wave's queries'
  int kend = r.len;
  if (r.causal) kend = min(kend, max(r.off + last + 1, r.pre));
  Visit visit = {kend > 0 ? (kend + TILE - 1) / TILE : 0};
  const int4* ranges = g.ranges ? g.ranges + qb.b * g.granules : nullptr;
  if (ranges != nullptr) {
    const int p = r.off + qb.q0, pt = r.off + tile * TILE;
    const bool inside = (p & 31) != 0;
    DocRange block = {0x7fffffff, 0}, own = block;
#pragma unroll
    for (int j = 0; j < ATT_ROWS / 32 + 1; j++) {
      const int4 e = granule_at(ranges, g.granules, j < ATT_ROWS / 32 || inside ? (p >> 5) + j : -1);
      block = {min(block.lo, e.x), max(block.hi, e.y)};
    }
#pragma unroll
    for (int j = 0; j < 3; j++) {
      const int4 e = granule_at(ranges, g.granules, j < 2 || inside ? (pt >> 5) + j : -1);
      own = {min(own.lo, e.x), max(own.hi, e.y)};
    }
    for (int w = 0; w * 64 < visit.to; w++) {
      const int t = w * 64 + lane;
      DocRange keys = {0x7fffffff, 0}, all = keys;  // of the tile, and of its key block of ATT_ROWS
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int4 e = granule_at(ranges, g.granules, (t >> 1) * 4 + j);
        all = {min(all.lo, e.x), max(all.hi, e.y)};
        if ((j >> 1) == (t & 1)) keys = {min(keys.lo, e.x), max(keys.hi, e.y)};
      }
      const uint64_t word = __ballot(t < visit.to && block.meets(keys)), wrote = __ballot(t < visit.to && own.meets(all));
      if (lane == 0) {
        if (w % WAVES == wave) bits[w] = word;
        halves[wave][w] = halves[wave][ATT_WORDS + w] = wrote;
      }
    }
    visit.bits = bits;
    visit.half = halves[wave];
    __syncthreads();
  }
  const int count = visit_count(visit);
  visit.start(0);
  int cur = visit.next(), alike = visit.alike, nxt = visit.next();
  auto copy = [&](int t, u16* K, u16* S) __attribute__((always_inline)) {
    dma.copy(K, kbase, t * TILE, r.len, wave);
    const u16* m = sbase + (int64_t)min(t, g.key_tiles - 1) * (TILE * ATT_ROWS) + wave * 2048;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)m, (short)0, 4096, 0x00020000);
#pragma unroll
    for (int p = 0; p < 4; p++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)((char*)S + wave * 4096 + p * 1024), 16, p * 1024 + sv[p & 1], 0, 0, 0);
  };
  auto step = [&](const u16* Kc, const u16* Sc, u16* Kn, u16* Sn) __attribute__((always_inline)) {
    copy(nxt, Kn, Sn);
    const int k0 = (cur >> 1) * ATT_ROWS;
    const int first = r.causal && k0 >= r.pre ? max(0, k0 - r.off) / TILE : 0;
    if ((alike & 1) && tile >= first && tile * TILE < r.t_q) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const u16x8 b = columns(Sc, c);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) acc[dt] = T::mfma32(ad.transposed(Kc, 16 * c, dt), b, acc[dt]);
      }
    }
    __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
    __syncthreads();
    cur = nxt;
    alike = visit.alike;
    nxt = visit.next();
  };
  if (count > 0) {
    copy(cur, K0, S0);
    __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
    __syncthreads();
    int it = 0;
    for (; it + 1 < count; it += 2) {
      step(K0, S0, K1, S1);
      step(K1, S1, K0, S0);
    }
    if (it < count) step(K0, S0, K1, S1);
  }
  const bool odd = any_odd(acc);  // a barrier: the tile buffers become staging below
  if (threadIdx.x == 0) g.odd[qb.bh * qb.nqb + qb.q0 / ATT_ROWS] = odd;
  u16* stage = wave == 0 ? K0 : wave == 1 ? K1 : wave == 2 ? S0 : S1;
  store_rows<T, D>(g.o0 + qb.bh * (int64_t)r.t_q * g.hd, acc, qb.wq0, r.t_q, g.hd, g.scale * ds_down<T>(), stage);
#endif
}

// ---- launches -------------------------------------------------------------------------------------------

enum AttendPass { ATTEND_PASS_FWD, ATTEND_PASS_DQ, ATTEND_PASS_DKV };

template <AttendPass PASS, typename T, int D, Cap CAP, bool BIAS>
int launch_fast_as(const FastArgs& g, const RuleArgs& ra, hipStream_t stream) {
  const int64_t blocks = PASS == ATTEND_PASS_DKV ? att_grid(g.batch * g.kv_heads, (ra.t_k + ATT_ROWS - 1) / ATT_ROWS, g.head_group)
                                                 : att_grid(g.batch * g.heads, (ra.t_q + ATT_ROWS - 1) / ATT_ROWS, g.head_group);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "attend: %lld workgroups exceed one launch", (long long)blocks);
  const dim3 grid((unsigned)blocks, PASS == ATTEND_PASS_DKV ? (unsigned)(g.head_parts * g.tile_parts) : 1), block(THREADS);
  if constexpr (PASS == ATTEND_PASS_DQ && D > 64) {
    if (g.ds != nullptr) {
      hipLaunchKernelGGL((attend_dq_handed<T, D>), grid, block, 0, stream, g, ra);
      return check_hip(hipGetLastError(), "launching attention");
    }
  }
  if constexpr (PASS == ATTEND_PASS_FWD && D > 64)
    hipLaunchKernelGGL((attend_fwd_wide<T, D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  else if constexpr (PASS == ATTEND_PASS_DQ && D > 64)
    hipLaunchKernelGGL((attend_dq_wide<T, D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  else if constexpr (PASS == ATTEND_PASS_FWD)
    hipLaunchKernelGGL((attend_fwd_mfma<T, D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  else if constexpr (PASS == ATTEND_PASS_DQ)
    hipLaunchKernelGGL((attend_dq_mfma<T, D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  else if constexpr (D <= 64)
    hipLaunchKernelGGL((attend_dkv_mfma<T, D, CAP, BIAS>), grid, block, 0, stream, g, ra);
  else if (g.ds != nullptr)
    hipLaunchKernelGGL((attend_dkv_wide<T, D, CAP, BIAS, true>), grid, dim3(64 * KV_WAVES), 0, stream, g, ra);
  else
    hipLaunchKernelGGL((attend_dkv_wide<T, D, CAP, BIAS, false>), grid, dim3(64 * KV_WAVES), 0, stream, g, ra);
  return check_hip(hipGetLastError(), "launching attention");
}

template <AttendPass PASS, typename T, int D>
int launch_fast_rules(const FastArgs& g, const RuleArgs& ra, hipStream_t stream) {
  const bool bias = ra.slopes != nullptr;
  if (ra.softcap > CAP_SHORT_MOST) return launch_fast_as<PASS, T, D, CAP_EXACT, true>(g, ra, stream);  // slopes of 0 without any
  if (ra.softcap > 0.f) return bias ? launch_fast_as<PASS, T, D, CAP_SHORT, true>(g, ra, stream) : launch_fast_as<PASS, T, D, CAP_SHORT, false>(g, ra, stream);
  return bias ? launch_fast_as<PASS, T, D, CAP_NONE, true>(g, ra, stream) : launch_fast_as<PASS, T, D, CAP_NONE, false>(g, ra, stream);
}

}  // namespace
}  // namespace limn
