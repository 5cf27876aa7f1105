// The head's cross entropy on 16-bit matrix cores: bf16/f16, width a multiple of 8, 16-byte aligned operands.
//
// Four products, each on the tiles and the LDS pipeline of matmul.hip (256 x 256 tiles by 8 waves, or 128 x 128 by
// 4 where the larger would leave compute units idle; operands from memory straight into swizzled LDS, the
// next 64 of k in flight while the current are multiplied):
//  - forward: logits = x w^T, never stored. A wave's accumulators hold 64 columns of 128 (64) rows; each row's
//    largest logit and the sum of exponentials over the tile's columns are found in registers, joined over
//    the tile's waves in LDS, and stored: 8 bytes a row and tile of 256 (128) columns. A second kernel joins the
//    tiles of a row in a fixed order. Bound by the matrix cores (2 rows width vocab operations).
//  - backward, a piece of the vocabulary at a time: the logits again, turned in the accumulators into
//    dz = g (exp(z - lse) - [v = target]) and stored once as the half-width operand it becomes; then
//    dx += dz w (float32 totals over the pieces, rounded once behind the last) and dw = dz^T x.
//    The piece (at most PIECE_BYTES of dz) is small enough that both products find most of it in the 256 MiB
//    last-level cache.
// Keeping the logits would save the second x w^T, a quarter of the matrix work, for rows * vocab * 4 bytes.
//
// A row without a target has dz = 0; what its x holds reaches nothing (see Products and the flags of xent_dz).

#include "matmul_dma.h"
#include "xent.h"

namespace limn {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int64_t PIECE_BYTES = (int64_t)128 << 20;

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; i++) z[i] = 0.f;
  return z;
}

__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- one tile's product, as matmul_dma computes it ----------------------------------------------------------

template <int BM>
struct Tile {
  static constexpr int WAVES = DmaTile<BM>::WAVES, WN = DmaTile<BM>::WN;
  static constexpr int WTM = BM / 2, WTN = BM / WN, TM = WTM / 32, TN = WTN / 32, KS = BK / 16;
  static_assert(WTN == 64, "a wave owns 64 columns");
};

#if defined(__HIP_DEVICE_COMPILE__)  // what the host pass, which only needs the kernels' stubs, cannot instantiate

// The last stage of a k-contiguous operand whose depth is no multiple of 64: chunks past it read as zeros
// (elsewhere they are the next row's elements).
template <int WAVES, typename D>
__device__ __forceinline__ void copy_last(const D& d, char* tile, int st, int depth, int wave, int lane) {
  const int64_t off = (d.first + st) * d.step, left = d.extent - off;
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(d.base + off), (short)0, (int)(left > 0 ? left : 0), 0x00020000);
  const int live = depth - (int)(d.first + st) * BK;  // elements of this stage that are there
#pragma unroll
  for (int q = 0; q < D::PASSES; q++) {
    const int row = (q * WAVES + wave) * D::RPI + lane / (D::RB / 16), c = (lane % (D::RB / 16)) ^ D::swizzle(row);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(tile + (q * WAVES + wave) * 1024), 16, c * 8 < live ? d.voff[q] : 0x7ffffff0, 0, 0, 0);
  }
}

// acc = sum over `stages` stages of k; `depth`: the depth at which k-contiguous operands end (TAIL). fix(tile of
// b, stage) runs between a stage's arrival and its first read, with a barrier before it and, if it returns true, behind it.
template <typename T, int BM, bool A_K, bool B_K, bool TAIL, typename DA, typename DB, typename FIX>
__device__ __forceinline__ void tile_product(const DA& da, const DB& db, char* A0, char* A1, char* B0, char* B1, int stages, int depth, int wave, int lane,
                                             f32x16 (*acc)[Tile<BM>::TN], FIX fix) {
  using L = Tile<BM>;
  constexpr int TM = L::TM, TN = L::TN, KS = L::KS;
  const int wm = wave / L::WN, wn = wave % L::WN;
  int rda[A_K ? KS : TM], rdb[B_K ? KS : TN];
  da.template offsets<TM>(wm * L::WTM, lane, rda);
  db.template offsets<TN>(wn * L::WTN, lane, rdb);
  u16x8 av[2][TM], bv[2][TN];
  auto read = [&](const char* at, const char* bt, int kk, u16x8* ao, u16x8* bo) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; i++) ao[i] = da.operand(at, rda, i, kk);
#pragma unroll
    for (int j = 0; j < TN; j++) bo[j] = db.operand(bt, rdb, j, kk);
  };
  auto copy = [&](char* at, char* bt, int st) __attribute__((always_inline)) {
    if constexpr (TAIL) {
      if (st == stages - 1) {
        copy_last<L::WAVES>(da, at, st, depth, wave, lane);
        copy_last<L::WAVES>(db, bt, st, depth, wave, lane);
        return;
      }
    }
    da.copy(at, st, wave);
    db.copy(bt, st, wave);
  };
  auto stage = [&](const char* at, const char* bt, char* an, char* bn, int st) __attribute__((always_inline)) {
    copy(an, bn, st + 1);
#pragma unroll
    for (int kk = 0; kk < KS; kk++) {
      const int p = kk & 1;
      if (kk + 1 < KS) read(at, bt, kk + 1, av[p ^ 1], bv[p ^ 1]);
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = T::mfma32(bv[p][j], av[p][i], acc[i][j]);
    }
    constexpr int RD = TM * DA::READS + TN * DB::READS, MF = TM * TN;
    if (!TAIL) __builtin_amdgcn_sched_group_barrier(0x020, DA::PASSES + DB::PASSES, 0);
#pragma unroll
    for (int kk = 0; kk < KS; kk++) {
      if (kk + 1 < KS) {
#pragma unroll
        for (int q = 0; q < (RD > MF ? RD : MF); q++) {
          if (q < MF) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (q < RD) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
      } else {
        __builtin_amdgcn_sched_group_barrier(0x008, MF, 0);
      }
    }
    __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
    __syncthreads();
    if (st + 1 < stages && fix(bn, st + 1)) __syncthreads();
    read(an, bn, 0, av[0], bv[0]);
  };
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = zero16();
  copy(A0, B0, 0);
  __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
  __syncthreads();
  if (fix(B0, 0)) __syncthreads();
  read(A0, B0, 0, av[0], bv[0]);
  for (int st = 0; st < stages; st += 2) {
    stage(A0, B0, A1, B1, st);
    if (st + 1 < stages) stage(A1, B1, A0, B0, st + 1);
  }
}

__device__ __forceinline__ bool no_fix(char*, int) { return false; }

#endif

// Which tile a workgroup takes: each XCD a contiguous run, in groups of 4 tile rows, as in matmul_dma.
__device__ __forceinline__ void tile_of(int64_t tiles_m, int64_t tiles_n, int64_t& tm, int64_t& tn, int64_t& slice) {
  int64_t id = blockIdx.x;
  if (gridDim.x % 8 == 0) id = (id % 8) * (gridDim.x / 8) + id / 8;
  const int64_t per = tiles_m * tiles_n;
  slice = id / per;
  const int64_t t = id - slice * per;
  constexpr int64_t GROUP = 4;
  const int64_t group = t / (GROUP * tiles_n), first = group * GROUP;
  const int64_t rows = tiles_m - first < GROUP ? tiles_m - first : GROUP;
  tm = first + (t - group * GROUP * tiles_n) % rows;
  tn = (t - group * GROUP * tiles_n) / rows;
}

struct Logits {
  const u16* x;
  const u16* w;         // the piece's rows
  const int* targets;
  int64_t rows, width, piece, vocab, v0;
  // forward
  float2* stats;        // (tiles of columns, rows): largest logit, sum of exponentials against it
  float* picked;        // (rows): the target's logit
  int64_t tile0;        // the piece's first tile
  // backward
  const float* lse;
  const float* g;
  u16* dz;              // (padded rows, ldz)
  int64_t ldz;
  int* flags;           // one a 64 rows: a row without a target has logits that are not finite
};

#define LIMN_XENT_LDS(BM)                                                          \
  using L = Tile<BM>;                                                              \
  constexpr int BYTES = BM * BK * 2;                                               \
  __shared__ __attribute__((aligned(1024))) char A0[BYTES];                        \
  __shared__ __attribute__((aligned(1024))) char A1[BYTES];                        \
  __shared__ __attribute__((aligned(1024))) char B0[BYTES];                        \
  __shared__ __attribute__((aligned(1024))) char B1[BYTES];                        \
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n32 = lane & 31; \
  const int wm = wave / L::WN, wn = wave % L::WN;

// ---- forward: a tile of logits into its rows' statistics ------------------------------------------------------

template <typename T, int BM, bool TAIL>
__global__ __launch_bounds__(64 * Tile<BM>::WAVES, 2) void xent_stats(Logits a) {
#if defined(__HIP_DEVICE_COMPILE__)
  LIMN_XENT_LDS(BM)
  const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.piece + BM - 1) / BM;
  int64_t tm, tn, slice;
  tile_of(tiles_m, tiles_n, tm, tn, slice);
  const int64_t m0 = tm * BM, n0 = tn * BM;
  const DmaOperand<BM, true, L::WAVES> da(a.x, a.rows, a.width, a.width, m0, 0, wave, lane), db(a.w, a.piece, a.width, a.width, n0, 0, wave, lane);
  f32x16 acc[L::TM][L::TN];
  tile_product<T, BM, true, true, TAIL>(da, db, A0, A1, B0, B1, (int)((a.width + BK - 1) / BK), (int)a.width, wave, lane, acc, no_fix);

  // lane: rows 32 i + n32 of the wave, columns 32 j + 8 q + 4 h + e in items 4 q + e
  const int64_t col0 = n0 + wn * 64;
  if (col0 + 64 > a.piece) {
#pragma unroll
    for (int j = 0; j < L::TN; j++)
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (col0 + 32 * j + 8 * (e >> 2) + 4 * h + (e & 3) >= a.piece) {
#pragma unroll
          for (int i = 0; i < L::TM; i++) acc[i][j][e] = -__builtin_inff();
        }
  }
  __syncthreads();
  float2* join = (float2*)A0;  // (WN, BM)
#pragma unroll
  for (int i = 0; i < L::TM; i++) {
    const int r = wm * L::WTM + 32 * i + n32;
    const int64_t row = m0 + r;
    float mx = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < L::TN; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) mx = fmaxf(mx, acc[i][j][e]);
    mx = pair_max(mx);
    const float base = mx == -__builtin_inff() ? 0.f : mx * LOG2E;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < L::TN; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) s += fast_exp2(fmaf(acc[i][j][e], LOG2E, -base));
    s = pair_sum(s);
    if (h == 0) join[wn * BM + r] = make_float2(mx, s);
    const int64_t t = row < a.rows ? (int64_t)a.targets[row] - a.v0 - col0 : -1;
    if (t >= 0 && t < 64 && (((int)t >> 2) & 1) == h) {  // this lane holds the target's logit
      float z = 0.f;
#pragma unroll
      for (int j = 0; j < L::TN; j++)
#pragma unroll
        for (int e = 0; e < 16; e++)
          if ((int)t == 32 * j + 8 * (e >> 2) + 4 * h + (e & 3)) z = acc[i][j][e];
      a.picked[row] = z;
    }
  }
  __syncthreads();
  for (int r = threadIdx.x; r < BM; r += 64 * L::WAVES) {
    if (m0 + r >= a.rows) continue;
    float top = -__builtin_inff(), total = 0.f;
#pragma unroll
    for (int w = 0; w < L::WN; w++) top = fmaxf(top, join[w * BM + r].x);
#pragma unroll
    for (int w = 0; w < L::WN; w++) {
      const float2 p = join[w * BM + r];
      total += p.x == -__builtin_inff() ? p.y : p.y * fast_exp2((p.x - top) * LOG2E);
    }
    a.stats[(a.tile0 + tn) * a.rows + m0 + r] = make_float2(top, total);
  }
#endif
}

// 32 rows a workgroup, 8 threads a row, each a run of the row's tiles; joined in order.
__global__ __launch_bounds__(256) void xent_rows(const float2* __restrict__ stats, const float* __restrict__ picked, const int* __restrict__ targets,
                                                 float* __restrict__ loss, float* __restrict__ lse, int64_t rows, int64_t tiles, int64_t vocab) {
  __shared__ float2 part[8][32];
  const int r = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t row = blockIdx.x * (int64_t)32 + r, run = (tiles + 7) / 8, t1 = (g + 1) * run < tiles ? (g + 1) * run : tiles;
  float m = -__builtin_inff(), l = 0.f;
  if (row < rows) {
#pragma unroll 4
    for (int64_t t = g * run; t < t1; t++) {
      const float2 p = stats[t * rows + row];
      const float top = fmaxf(m, p.x);
      if (top == -__builtin_inff()) {
        l += p.y;
      } else {
        l = l * fast_exp2((m - top) * LOG2E) + p.y * fast_exp2((p.x - top) * LOG2E);
      }
      m = top;
    }
  }
  part[g][r] = make_float2(m, l);
  __syncthreads();
  if (g == 0 && row < rows) {
    float top = -__builtin_inff(), total = 0.f;
    for (int k = 0; k < 8; k++) top = fmaxf(top, part[k][r].x);
    for (int k = 0; k < 8; k++) total += part[k][r].x == -__builtin_inff() ? part[k][r].y : part[k][r].y * fast_exp2((part[k][r].x - top) * LOG2E);
    const float z = top + logf(total);
    const int t = targets[row];
    lse[row] = z;
    loss[row] = t >= 0 && t < vocab ? z - picked[row] : 0.f;
  }
}

// ---- backward: a tile of logits into dz -------------------------------------------------------------------

template <typename T, int BM, bool TAIL>
__global__ __launch_bounds__(64 * Tile<BM>::WAVES, 2) void xent_dz(Logits a) {
#if defined(__HIP_DEVICE_COMPILE__)
  LIMN_XENT_LDS(BM)
  const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = a.ldz / BM;
  int64_t tm, tn, slice;
  tile_of(tiles_m, tiles_n, tm, tn, slice);
  const int64_t m0 = tm * BM, n0 = tn * BM;
  const DmaOperand<BM, true, L::WAVES> da(a.x, a.rows, a.width, a.width, m0, 0, wave, lane), db(a.w, a.piece, a.width, a.width, n0, 0, wave, lane);
  f32x16 acc[L::TM][L::TN];
  tile_product<T, BM, true, true, TAIL>(da, db, A0, A1, B0, B1, (int)((a.width + BK - 1) / BK), (int)a.width, wave, lane, acc, no_fix);

  const int64_t col0 = n0 + wn * 64;
  __syncthreads();
  // each wave writes its rows' halves through 8 KB of LDS, 64 rows at a time, and stores whole 128-byte
  // segments; rows past the end and columns past the piece are zeros, which both products count on
  int* odd = (int*)B1;  // (BM / 64): see flags
  if (threadIdx.x < BM / 64) odd[threadIdx.x] = 0;
  __syncthreads();
  char* const region = (wave < 4 ? A0 : A1) + (wave & 3) * (BM == 256 ? 8192 : 4096);
  constexpr int PASS = BM == 256 ? 2 : 1;  // 32-row blocks a pass
#pragma unroll
  for (int p = 0; p < L::TM / PASS; p++) {
#pragma unroll
    for (int ii = 0; ii < PASS; ii++) {
      const int i = p * PASS + ii;
      const int64_t row = m0 + wm * L::WTM + 32 * i + n32;
      const int t32 = row < a.rows ? a.targets[row] : -1;
      const bool live = t32 >= 0 && t32 < a.vocab;
      const int64_t t = (int64_t)t32 - a.v0 - col0;
      const float l2 = live ? a.lse[row] * LOG2E : 0.f, g = live ? a.g[row] : 0.f;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < L::TN; j++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int c = 32 * j + 8 * q + 4 * h + e;
            const float z = acc[i][j][4 * q + e];
            bad |= !(fabsf(z) <= 3.402823466e38f);
            const float d = g * (fast_exp2(fmaf(z, LOG2E, -l2)) - (c == t ? 1.f : 0.f));
            v[e] = live && col0 + c < a.piece ? d : 0.f;
          }
          const int r = ii * 32 + n32;
          *(uint2*)(region + r * 128 + ((4 * j + q) ^ ((r >> 1) & 7)) * 16 + 8 * h) = make_uint2(T::pack2(v[0], v[1]), T::pack2(v[2], v[3]));
        }
      if (bad && !live && row < a.rows) odd[(row - m0) / 64] = 1;  // every writer writes 1
    }
#pragma unroll
    for (int it = 0; it < PASS * 4; it++) {
      const int r = it * 8 + lane / 8, cc = lane & 7;
      const u32x4 s = *(const u32x4*)(region + r * 128 + (cc ^ ((r >> 1) & 7)) * 16);
      *(u32x4*)(a.dz + (m0 + wm * L::WTM + p * PASS * 32 + r) * a.ldz + col0 + cc * 8) = s;
    }
  }
  if (tn == 0) {
    __syncthreads();
    if (threadIdx.x < BM / 64) a.flags[m0 / 64 + threadIdx.x] = odd[threadIdx.x];
  }
#endif
}

// ---- backward: dx += dz w, dw = dz^T x ------------------------------------------------------------------------

// Products of dz: C (m, n) = sum_k A B with A dz (k-contiguous for dx, m-contiguous for dw), B the weights or the rows
// (n-contiguous), k cut into slices of `chunk`. A is padded with zeros to whole tiles; B's rows past b_depth
// read as zeros.
struct Products {
  const u16* a;
  const u16* b;
  int64_t m, n, k;       // of the result and of the padded contraction
  int64_t a_rows, a_depth, a_stride;
  int64_t b_depth, b_stride;
  int64_t chunk;
  u16* out;              // of half width, row stride n; or nullptr:
  float* wide;           // (slices, m, n) float32
  const float* add;      // (m, n) float32 added to an unsplit result, or nullptr
  const int* flags;      // dw: see xent_dz; a flagged stage's rows of x without a target are taken as zeros
  const int* targets;
  int64_t rows, vocab;
};

template <typename T, int BM, bool A_K>
__global__ __launch_bounds__(64 * Tile<BM>::WAVES, 2) void xent_product(Products s) {
#if defined(__HIP_DEVICE_COMPILE__)
  LIMN_XENT_LDS(BM)
  const int64_t tiles_m = (s.m + BM - 1) / BM, tiles_n = (s.n + BM - 1) / BM;
  int64_t tm, tn, slice;
  tile_of(tiles_m, tiles_n, tm, tn, slice);
  const int64_t m0 = tm * BM, n0 = tn * BM, k_lo = slice * s.chunk, k_hi = k_lo + s.chunk < s.k ? k_lo + s.chunk : s.k;
  const DmaOperand<BM, A_K, L::WAVES> da(s.a, s.a_rows, s.a_depth, s.a_stride, m0, k_lo, wave, lane);
  const DmaOperand<BM, false, L::WAVES> db(s.b, s.n, s.b_depth, s.b_stride, n0, k_lo, wave, lane);
  f32x16 acc[L::TM][L::TN];
  // an infinity or a NaN in a row of x without a target meets a dz of 0, which would be NaN: such rows of the
  // tile are overwritten with zeros (only where xent_dz saw one; a scalar load a stage otherwise)
  auto fix = [&](char* tile, int st) __attribute__((always_inline)) {
    if (A_K) return false;
    const int64_t row0 = k_lo + (int64_t)st * BK;
    if (row0 >= s.rows || s.flags[row0 / 64] == 0) return false;
    constexpr int RB = BM * 2, PER = 64 * L::WAVES / BK;  // bytes an LDS row of k, threads a row
    const int r = threadIdx.x / PER;
    const int t = row0 + r < s.rows ? s.targets[row0 + r] : -1;
    if (t < 0 || t >= s.vocab)
      for (int c = threadIdx.x % PER; c < RB / 16; c += PER) *(u32x4*)(tile + r * RB + c * 16) = u32x4{0, 0, 0, 0};
    return true;
  };
  tile_product<T, BM, A_K, false, false>(da, db, A0, A1, B0, B1, (int)((k_hi - k_lo + BK - 1) / BK), 0, wave, lane, acc, fix);

  __syncthreads();
  // 32 rows x 64 columns of float32 a wave through LDS (8 KB), then whole row segments
  char* const region = (wave < 4 ? A0 : A1) + (wave & 3) * 4096 + (BM == 256 ? (wave & 3) * 4096 : 0);
#pragma unroll
  for (int i = 0; i < L::TM; i++) {
    if (BM == 256) {
#pragma unroll
      for (int j = 0; j < L::TN; j++)
#pragma unroll
        for (int q = 0; q < 4; q++)
          *(f32x4*)(region + n32 * 256 + ((8 * j + 2 * q + h) ^ (n32 & 15)) * 16) = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    }
#pragma unroll
    for (int half = 0; half < (BM == 256 ? 1 : 2); half++) {
      if (BM != 256) {  // 4 KB a wave: 32 columns at a time
#pragma unroll
        for (int q = 0; q < 4; q++)
          *(f32x4*)(region + n32 * 128 + ((2 * q + h) ^ (n32 & 7)) * 16) =
              f32x4{acc[i][half][4 * q], acc[i][half][4 * q + 1], acc[i][half][4 * q + 2], acc[i][half][4 * q + 3]};
      }
      constexpr int CPR = BM == 256 ? 16 : 8, RPI = 64 / CPR;  // 16-byte chunks a staged row, rows an instruction
#pragma unroll
      for (int it = 0; it < 32 / RPI; it++) {
        const int r = it * RPI + lane / CPR, cc = lane % CPR;
        f32x4 v = *(const f32x4*)(region + r * CPR * 16 + (cc ^ (r & (CPR - 1))) * 16);
        const int64_t row = m0 + wm * L::WTM + 32 * i + r, col = n0 + wn * 64 + half * 32 + cc * 4;
        if (row >= s.m || col >= s.n) continue;  // n is a multiple of 8
        if (s.add != nullptr) v += *(const f32x4*)(s.add + row * s.n + col);
        if (s.out != nullptr)
          *(uint2*)(s.out + row * s.n + col) = make_uint2(T::pack2(v[0], v[1]), T::pack2(v[2], v[3]));
        else
          *(f32x4*)(s.wide + (slice * s.m + row) * s.n + col) = v;
      }
    }
  }
#endif
}

// out = round(add + slices in order), or the same kept in float32
template <typename T>
__global__ __launch_bounds__(256) void xent_fold(const float* __restrict__ slices, const float* add, int64_t count, int64_t total, u16* out, float* wide) {
  for (int64_t i = (blockIdx.x * (int64_t)256 + threadIdx.x) * 4; i < total; i += (int64_t)gridDim.x * 1024) {
    f32x4 v = *(const f32x4*)(slices + i);
    for (int64_t k = 1; k < count; k++) v += *(const f32x4*)(slices + k * total + i);
    if (add != nullptr) v += *(const f32x4*)(add + i);
    if (out != nullptr)
      *(uint2*)(out + i) = make_uint2(T::pack2(v[0], v[1]), T::pack2(v[2], v[3]));
    else
      *(f32x4*)(wide + i) = v;
  }
}

// ---- plans ------------------------------------------------------------------------------------------------

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

constexpr int64_t FILL = 256;  // workgroups that give every CU one

int tile_for(int64_t m, int64_t n) { return ((m + 255) / 256) * ((n + 255) / 256) >= FILL ? 256 : 128; }

// vocabulary entries whose dz goes by at a time, a multiple of 256
int64_t piece_of(const XentArgs& a) {
  const int64_t whole = up(a.vocab, 256), most = PIECE_BYTES / 2 / up(a.rows, 256) / 256 * 256;
  return most >= whole ? whole : most < 1024 ? 1024 : most;
}

struct Cut {
  int tile;
  int64_t split, chunk;
};
Cut cut(int64_t m, int64_t n, int64_t k) {
  const MatmulPlan p = plan_matmul(MatmulShape{1, m, n, k});
  return {p.tile, p.split, p.chunk};
}

struct BwdPlan {
  int64_t piece, pieces, rows_pad, slices;  // slices: float32 (slices x result) bytes the products need at most
};

int64_t product_bytes(int64_t m, int64_t n, int64_t k) {
  const Cut c = cut(m, n, k);
  return c.split > 1 ? c.split * m * n * 4 : 0;
}

BwdPlan bwd_plan(const XentArgs& a) {
  BwdPlan p;
  p.piece = piece_of(a);
  p.pieces = (a.vocab + p.piece - 1) / p.piece;
  p.rows_pad = up(a.rows, 256);
  p.slices = 0;
  for (const int64_t n : {p.piece < a.vocab ? p.piece : a.vocab, a.vocab - (p.pieces - 1) * p.piece}) {
    const int64_t dx = product_bytes(a.rows, a.width, up(n, 64)), dw = product_bytes(n, a.width, up(a.rows, 64));
    if (dx > p.slices) p.slices = dx;
    if (dw > p.slices) p.slices = dw;
  }
  return p;
}

// rows of a w piece whose byte offsets stay in 32 bits
int64_t stats_piece(const XentArgs& a) {
  const int64_t most = ((int64_t)0x70000000 / 2 / a.width) / 256 * 256;
  return most < a.vocab ? most : up(a.vocab, 256);
}

template <typename T, int BM>
int launch_stats(const Logits& l, hipStream_t stream) {
  const int64_t blocks = ((l.rows + BM - 1) / BM) * ((l.piece + BM - 1) / BM);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "xent: %lld workgroups exceed one launch", (long long)blocks);
  const dim3 grid((unsigned)blocks), block(64 * Tile<BM>::WAVES);
  if (l.width % BK == 0)
    hipLaunchKernelGGL((xent_stats<T, BM, false>), grid, block, 0, stream, l);
  else
    hipLaunchKernelGGL((xent_stats<T, BM, true>), grid, block, 0, stream, l);
  return check_hip(hipGetLastError(), "launching the cross entropy's logits");
}

template <typename T, int BM>
int launch_dz(const Logits& l, hipStream_t stream) {
  const int64_t blocks = ((l.rows + BM - 1) / BM) * (l.ldz / BM);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "xent: %lld workgroups exceed one launch", (long long)blocks);
  const dim3 grid((unsigned)blocks), block(64 * Tile<BM>::WAVES);
  if (l.width % BK == 0)
    hipLaunchKernelGGL((xent_dz<T, BM, false>), grid, block, 0, stream, l);
  else
    hipLaunchKernelGGL((xent_dz<T, BM, true>), grid, block, 0, stream, l);
  return check_hip(hipGetLastError(), "launching the cross entropy's gradient");
}

template <typename T, bool A_K>
int launch_product(Products s, const Cut& c, float* slices, float* acc, bool first, u16* out, hipStream_t stream) {
  // unsplit: straight to out (the last piece of dx, or dw), or into the float32 totals; split: slices, then a fold
  const bool split = c.split > 1;
  s.chunk = c.chunk;
  s.out = split ? nullptr : out;
  s.wide = split ? slices : acc;
  s.add = split || first ? nullptr : acc;
  const int64_t blocks = c.split * ((s.m + c.tile - 1) / c.tile) * ((s.n + c.tile - 1) / c.tile);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "xent: %lld workgroups exceed one launch", (long long)blocks);
  if (c.tile == 256)
    hipLaunchKernelGGL((xent_product<T, 256, A_K>), dim3((unsigned)blocks), dim3(512), 0, stream, s);
  else
    hipLaunchKernelGGL((xent_product<T, 128, A_K>), dim3((unsigned)blocks), dim3(256), 0, stream, s);
  const int rc = check_hip(hipGetLastError(), "launching a product of the cross entropy's gradient");
  if (rc != LIMN_HIP_OK || !split) return rc;
  const int64_t total = s.m * s.n, groups = (total / 4 + 255) / 256;
  hipLaunchKernelGGL((xent_fold<T>), dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(256), 0, stream, slices, first ? nullptr : acc, c.split, total, out, acc);
  return check_hip(hipGetLastError(), "launching the fold of a product's slices");
}

template <typename T>
int fwd(const XentArgs& a) {
  const int64_t piece = stats_piece(a);
  const int bm = tile_for(a.rows, a.vocab);
  XentSpace space(a.workspace);
  const int64_t tiles = (a.vocab + bm - 1) / bm;
  Logits l = {};
  l.x = (const u16*)a.x, l.targets = a.targets, l.rows = a.rows, l.width = a.width, l.vocab = a.vocab;
  l.stats = (float2*)space.take(tiles * a.rows * 8);
  l.picked = (float*)space.take(a.rows * 4);
  int rc = LIMN_HIP_OK;
  for (int64_t v0 = 0; v0 < a.vocab && rc == LIMN_HIP_OK; v0 += piece) {
    l.w = (const u16*)a.w + v0 * a.width;
    l.v0 = v0;
    l.piece = a.vocab - v0 < piece ? a.vocab - v0 : piece;
    l.tile0 = v0 / bm;
    rc = bm == 256 ? launch_stats<T, 256>(l, a.stream) : launch_stats<T, 128>(l, a.stream);
  }
  if (rc != LIMN_HIP_OK) return rc;
  hipLaunchKernelGGL(xent_rows, dim3((unsigned)((a.rows + 31) / 32)), dim3(256), 0, a.stream, l.stats, l.picked, a.targets, (float*)a.o0, (float*)a.o1, a.rows, tiles,
                     a.vocab);
  return check_hip(hipGetLastError(), "launching the cross entropy's rows");
}

template <typename T>
int bwd(const XentArgs& a) {
  const BwdPlan p = bwd_plan(a);
  XentSpace space(a.workspace);
  Logits l = {};
  l.x = (const u16*)a.x, l.targets = a.targets, l.rows = a.rows, l.width = a.width, l.vocab = a.vocab, l.lse = a.lse_in, l.g = a.g;
  l.dz = (u16*)space.take(p.rows_pad * p.piece * 2);
  l.flags = (int*)space.take(p.rows_pad / 64 * 4);
  float* slices = (float*)space.take(p.slices);
  float* acc = p.pieces > 1 ? (float*)space.take(a.rows * a.width * 4) : nullptr;
  for (int64_t v0 = 0; v0 < a.vocab; v0 += p.piece) {
    const bool first = v0 == 0, last = v0 + p.piece >= a.vocab;
    l.w = (const u16*)a.w + v0 * a.width;
    l.v0 = v0;
    l.piece = last ? a.vocab - v0 : p.piece;
    l.ldz = up(l.piece, 256);
    int rc = tile_for(a.rows, l.ldz) == 256 ? launch_dz<T, 256>(l, a.stream) : launch_dz<T, 128>(l, a.stream);
    if (rc != LIMN_HIP_OK) return rc;
    Products s = {};
    s.rows = a.rows, s.vocab = a.vocab, s.targets = a.targets, s.flags = l.flags;
    s.a = l.dz, s.b = l.w, s.m = a.rows, s.n = a.width, s.k = up(l.piece, 64);
    s.a_rows = p.rows_pad, s.a_depth = l.ldz, s.a_stride = l.ldz, s.b_depth = l.piece, s.b_stride = a.width;
    rc = launch_product<T, true>(s, cut(s.m, s.n, s.k), slices, acc, first, last ? (u16*)a.o0 : nullptr, a.stream);
    if (rc != LIMN_HIP_OK) return rc;
    s.b = (const u16*)a.x, s.m = l.piece, s.k = up(a.rows, 64);
    s.a_rows = l.ldz, s.a_depth = p.rows_pad, s.b_depth = a.rows;
    rc = launch_product<T, false>(s, cut(s.m, s.n, s.k), slices, nullptr, true, (u16*)a.o1 + v0 * a.width, a.stream);
    if (rc != LIMN_HIP_OK) return rc;
  }
  return LIMN_HIP_OK;
}

}  // namespace

// 16-byte rows, every operand's bytes within 32-bit offsets of a base (a tile may reach 256 rows past its end)
bool xent_half_sizes(const XentArgs& a) {
  if (a.dtype == LIMN_HIP_FLOAT32 || a.width % 8 != 0) return false;
  const int64_t most = (int64_t)0x7f000000 / 2, piece = piece_of(a);
  if ((a.rows + 512) * a.width >= most || (stats_piece(a) + 512) * a.width >= most || stats_piece(a) < 256) return false;
  return (up(a.rows, 256) + 512) * piece < most && (piece + 512) * a.width < most;
}

int64_t xent_half_workspace(const XentArgs& a, bool backward) {
  if (!backward) return xent_align(((a.vocab + 127) / 128) * a.rows * 8) + xent_align(a.rows * 4);
  const BwdPlan p = bwd_plan(a);
  return xent_align(p.rows_pad * p.piece * 2) + xent_align(p.rows_pad / 64 * 4) + xent_align(p.slices) + (p.pieces > 1 ? xent_align(a.rows * a.width * 4) : 0);
}

int launch_xent_half_fwd(const XentArgs& a) { return a.dtype == LIMN_HIP_BFLOAT16 ? fwd<BF16>(a) : fwd<F16>(a); }
int launch_xent_half_bwd(const XentArgs& a) { return a.dtype == LIMN_HIP_BFLOAT16 ? bwd<BF16>(a) : bwd<F16>(a); }

}  // namespace limn
