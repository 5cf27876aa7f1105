// The head's cross entropy on 16-bit matrix cores.
//
// bf16 and f16 operands go as they are, or, where their rows are not 16-byte aligned or the width is no multiple of
// 8, from copies padded with zeros. float32 operands go as three bf16 parts each, x = h + m + l with h the
// nearest bf16 to x, m to x - h, l to the rest (8 + 8 + 8 bits and the parts' signs: x to 2^-24 or better, down to
// half of bf16's least step, 2^-134), and a
// product of two numbers as the six products of parts that are not below 2^-24 of it: h h, h m, m h, m m, h l, l h,
// the smallest first (the splitting published as BF16x6: Henry, Tang, Heinecke, Leveraging the bfloat16
// artificial intelligence datatype for higher-precision computations, 2019). 6 products at the 16-bit rate are
// 2.6 times as fast as one at the float32 matrix rate (157 TFLOP/s); the sums are float32 either way.
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
// 8192 rows x 2048 x 65536 bf16: 7.5-7.8 ms, the four products at 1130-1180 TFLOP/s (a library product reaches 1230); 2048 x
// 512 x 8191 float32: 473-500 us, 140 TFLOP/s in float32 terms (a library product 153); 48 rows x 512 x 32000 bf16: 68 us of kernels
// whose chains of stages few rows do not hide.
// Keeping the logits would save the second x w^T, a quarter of the matrix work, for rows * vocab * 4 bytes.
//
// Every operand is PARTS matrices of one shape, one part_a or part_b elements behind another (1 or 3).
//
// A row without a target has dz = 0; what its x holds reaches nothing (see Products and the flags of xent_dz), and its dx is
// stored as zeros, as a dz of 0 times a weight that is not finite would be NaN.

#include "matmul_dma.h"
#include "xent.h"

namespace limn {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int64_t PIECE_BYTES = (int64_t)128 << 20;

template <typename T>
constexpr bool IS_F16 = std::is_same<T, F16>::value;

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

// The operand copy of DmaOperand from `shift` bytes on; last: the stage at which a k-contiguous operand's depth
// ends, whose chunks past it read as zeros (elsewhere they are the next row's elements).
template <int WAVES, typename D>
__device__ __forceinline__ void copy_from(const D& d, int64_t shift, char* tile, int st, int wave) {
  const int64_t off = (d.first + st) * d.step, left = d.extent - off;
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(d.base + shift + off), (short)0, (int)(left > 0 ? left : 0), 0x00020000);
#pragma unroll
  for (int q = 0; q < D::PASSES; q++)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(tile + (q * WAVES + wave) * 1024), 16, d.voff[q], 0, 0, 0);
}
template <int WAVES, typename D>
__device__ __forceinline__ void copy_last(const D& d, int64_t shift, char* tile, int st, int depth, int wave, int lane) {
  const int64_t off = (d.first + st) * d.step, left = d.extent - off;
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(d.base + shift + off), (short)0, (int)(left > 0 ? left : 0), 0x00020000);
  const int live = depth - (int)(d.first + st) * BK;  // elements of this stage that are there
#pragma unroll
  for (int q = 0; q < D::PASSES; q++) {
    const int row = (q * WAVES + wave) * D::RPI + lane / (D::RB / 16), c = (lane % (D::RB / 16)) ^ D::swizzle(row);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(tile + (q * WAVES + wave) * 1024), 16, c * 8 < live ? d.voff[q] : 0x7ffffff0, 0, 0, 0);
  }
}

// acc = sum over `depth_stages` stages of k, for every pair of parts in turn, the smallest products first; `depth`:
// where k-contiguous operands end (TAIL). fix(tile of b, stage) runs between a stage's arrival and its first
// read, with a barrier before it and, if it returns true, behind it.
template <typename T, int BM, int PARTS, bool A_K, bool B_K, bool TAIL, typename DA, typename DB, typename FIX>
__device__ __forceinline__ void tile_product(const DA& da, const DB& db, int64_t part_a, int64_t part_b, char* A0, char* A1, char* B0, char* B1,
                                             int depth_stages, int depth, int wave, int lane, f32x16 (*acc)[Tile<BM>::TN], FIX fix) {
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
  // stages are copied in order: `at` is the next one's place in its pair of parts, `pair` the pair
  int at = 0, pair = 0;
  const int stages = PARTS == 3 ? 6 * depth_stages : depth_stages;
  auto copy = [&](char* an, char* bn) __attribute__((always_inline)) {
    // l h, h l, m m, m h, h m, h h: four bits a pair, the first lowest
    const int64_t sa = PARTS == 3 ? ((0x001102 >> (4 * pair)) & 15) * part_a * 2 : 0, sb = PARTS == 3 ? ((0x010120 >> (4 * pair)) & 15) * part_b * 2 : 0;
    bool done = false;
    if constexpr (TAIL) {
      if (at == depth_stages - 1) {
        copy_last<L::WAVES>(da, sa, an, at, depth, wave, lane);
        copy_last<L::WAVES>(db, sb, bn, at, depth, wave, lane);
        done = true;
      }
    }
    if (!done) {
      copy_from<L::WAVES>(da, sa, an, at, wave);
      copy_from<L::WAVES>(db, sb, bn, at, wave);
    }
    at++;
    if (PARTS == 3 && at == depth_stages && pair < 5) at = 0, pair++;
  };
  auto stage = [&](const char* at_, const char* bt, char* an, char* bn, int st) __attribute__((always_inline)) {
    const int coming = at;
    copy(an, bn);
#pragma unroll
    for (int kk = 0; kk < KS; kk++) {
      const int p = kk & 1;
      if (kk + 1 < KS) read(at_, bt, kk + 1, av[p ^ 1], bv[p ^ 1]);
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
    if (st + 1 < stages && fix(bn, coming)) __syncthreads();
    read(an, bn, 0, av[0], bv[0]);
  };
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = zero16();
  copy(A0, B0);
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
  int64_t part_x, part_w;  // elements between the parts
  // forward
  float2* stats;        // (tiles of columns, rows): largest logit, sum of exponentials against it
  float* picked;        // (rows): the target's logit
  int64_t tile0;        // the piece's first tile
  // backward
  const float* lse;
  const float* g;
  u16* dz;              // (PARTS, padded rows, ldz)
  int64_t ldz, part_dz;
  int* flags;           // one a 64 rows: a row without a target has logits that are not finite
  const float* scale;   // float16: what dz is multiplied by, and its inverse
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

template <typename T, int BM, int PARTS, bool TAIL>
__global__ __launch_bounds__(64 * Tile<BM>::WAVES, 2) void xent_stats(Logits a) {
#if defined(__HIP_DEVICE_COMPILE__)
  LIMN_XENT_LDS(BM)
  const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.piece + BM - 1) / BM;
  int64_t tm, tn, slice;
  tile_of(tiles_m, tiles_n, tm, tn, slice);
  const int64_t m0 = tm * BM, n0 = tn * BM;
  const DmaOperand<BM, true, L::WAVES> da(a.x, a.rows, a.width, a.width, m0, 0, wave, lane), db(a.w, a.piece, a.width, a.width, n0, 0, wave, lane);
  f32x16 acc[L::TM][L::TN];
  tile_product<T, BM, PARTS, true, true, TAIL>(da, db, a.part_x, a.part_w, A0, A1, B0, B1, (int)((a.width + BK - 1) / BK), (int)a.width, wave, lane, acc, no_fix);

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

// R rows a workgroup, 256 / R threads a row, each a run of the row's tiles; joined in order. Bound by the latency of a
// thread's chain of loads: 32 rows where that gives every CU a workgroup, else 4 (48 rows, 250 tiles: 13 -> 5.5 us).
template <int R>
__global__ __launch_bounds__(256) void xent_rows(const float2* __restrict__ stats, const float* __restrict__ picked, const int* __restrict__ targets,
                                                 float* __restrict__ loss, float* __restrict__ lse, int64_t rows, int64_t tiles, int64_t vocab) {
  constexpr int RUNS = 256 / R;
  __shared__ float2 part[RUNS][R];
  const int r = threadIdx.x % R, g = threadIdx.x / R;
  const int64_t row = blockIdx.x * (int64_t)R + r, run = (tiles + RUNS - 1) / RUNS, t1 = (g + 1) * run < tiles ? (g + 1) * run : tiles;
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
    for (int k = 0; k < RUNS; k++) top = fmaxf(top, part[k][r].x);
    for (int k = 0; k < RUNS; k++) total += part[k][r].x == -__builtin_inff() ? part[k][r].y : part[k][r].y * fast_exp2((part[k][r].x - top) * LOG2E);
    const float z = top + logf(total);
    const int t = targets[row];
    lse[row] = z;
    loss[row] = t >= 0 && t < vocab ? z - picked[row] : 0.f;
  }
}

// dz = g (p - [v = target]) can lie far below float16's numbers where g is a mean's 1 / rows and p one of many: it goes
// multiplied by the power of two that brings the largest |g| (of the finite ones with a target) to [2^14, 2^15), which
// the products' stores take off again. One workgroup; {power, inverse}.
__global__ __launch_bounds__(1024) void xent_scale(const float* __restrict__ g, const int* __restrict__ targets, int64_t rows, int64_t vocab, float* __restrict__ scale) {
  __shared__ float most[16];
  float m = 0.f;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < rows; r += 1024) {
    const float v = fabsf(g[r]);
    const int t = targets[r];
    if (t >= 0 && t < vocab && v <= 3.402823466e38f) m = fmaxf(m, v);
  }
#pragma unroll
  for (int d = 32; d > 0; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; i++) m = fmaxf(m, most[i]);
  const int bits = m == 0.f ? 0 : 14 - ilogbf(m);
  const int e = bits < 120 ? bits : 120;  // the inverse stays a normal number
  scale[0] = ldexpf(1.f, e);
  scale[1] = ldexpf(1.f, -e);
}

// ---- backward: a tile of logits into dz -------------------------------------------------------------------

template <typename T, int BM, int PARTS, bool TAIL>
__global__ __launch_bounds__(64 * Tile<BM>::WAVES, 2) void xent_dz(Logits a) {
#if defined(__HIP_DEVICE_COMPILE__)
  LIMN_XENT_LDS(BM)
  const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = a.ldz / BM;
  int64_t tm, tn, slice;
  tile_of(tiles_m, tiles_n, tm, tn, slice);
  const int64_t m0 = tm * BM, n0 = tn * BM;
  const DmaOperand<BM, true, L::WAVES> da(a.x, a.rows, a.width, a.width, m0, 0, wave, lane), db(a.w, a.piece, a.width, a.width, n0, 0, wave, lane);
  f32x16 acc[L::TM][L::TN];
  tile_product<T, BM, PARTS, true, true, TAIL>(da, db, a.part_x, a.part_w, A0, A1, B0, B1, (int)((a.width + BK - 1) / BK), (int)a.width, wave, lane, acc, no_fix);

  const int64_t col0 = n0 + wn * 64;
  const float up = IS_F16<T> ? a.scale[0] : 1.f;
  __syncthreads();
  // each wave writes its rows' halves through 8 KB of LDS, 64 rows at a time, and stores whole 128-byte
  // segments; rows past the end and columns past the piece are zeros, which both products count on
  int* odd = (int*)B1;  // (BM / 64): see flags
  if (threadIdx.x < BM / 64) odd[threadIdx.x] = 0;
  __syncthreads();
  char* const region = (wave < 4 ? A0 : A1) + (wave & 3) * (BM == 256 ? 8192 : 4096);
  constexpr int PASS = BM == 256 ? 2 : 1;  // 32-row blocks a pass
#pragma unroll
  for (int i = 0; i < L::TM; i++) {
    const int64_t row = m0 + wm * L::WTM + 32 * i + n32;
    const int t32 = row < a.rows ? a.targets[row] : -1;
    const bool live = t32 >= 0 && t32 < a.vocab;
    const int64_t t = (int64_t)t32 - a.v0 - col0;
    const float l2 = live ? a.lse[row] * LOG2E : 0.f, g = live ? a.g[row] * up : 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < L::TN; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int c = 32 * j + 8 * (e >> 2) + 4 * h + (e & 3);
        const float z = acc[i][j][e];
        bad |= !(fabsf(z) <= 3.402823466e38f);
        const float d = g * (fast_exp2(fmaf(z, LOG2E, -l2)) - (c == t ? 1.f : 0.f));
        acc[i][j][e] = live && col0 + c < a.piece ? d : 0.f;
      }
    if (bad && !live && row < a.rows) odd[(row - m0) / 64] = 1;  // every writer writes 1
  }
#pragma unroll
  for (int part = 0; part < PARTS; part++) {
#pragma unroll
    for (int p = 0; p < L::TM / PASS; p++) {
#pragma unroll
      for (int ii = 0; ii < PASS; ii++) {
        const int i = p * PASS + ii, r = ii * 32 + n32;
#pragma unroll
        for (int j = 0; j < L::TN; j++)
#pragma unroll
          for (int q = 0; q < 4; q++) {
            uint2 w;
            w.x = T::pack2(acc[i][j][4 * q], acc[i][j][4 * q + 1]);
            w.y = T::pack2(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
            if (part + 1 < PARTS) {  // what is left for the next part
              acc[i][j][4 * q] -= T::unpack((u16)w.x);
              acc[i][j][4 * q + 1] -= T::unpack((u16)(w.x >> 16));
              acc[i][j][4 * q + 2] -= T::unpack((u16)w.y);
              acc[i][j][4 * q + 3] -= T::unpack((u16)(w.y >> 16));
            }
            *(uint2*)(region + r * 128 + ((4 * j + q) ^ ((r >> 1) & 7)) * 16 + 8 * h) = w;
          }
      }
#pragma unroll
      for (int it = 0; it < PASS * 4; it++) {
        const int r = it * 8 + lane / 8, cc = lane & 7;
        const u32x4 s = *(const u32x4*)(region + r * 128 + (cc ^ ((r >> 1) & 7)) * 16);
        *(u32x4*)(a.dz + part * a.part_dz + (m0 + wm * L::WTM + p * PASS * 32 + r) * a.ldz + col0 + cc * 8) = s;
      }
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
  int64_t b_depth, b_stride, b_cols;
  int64_t part_a, part_b;
  int64_t chunk;
  int64_t width;         // columns of the result that there are: n rounds them up to a multiple of 8
  void* out;             // (m, width) of the result's type; or nullptr:
  int out_f32, vec;      // its type; whether its rows take vector stores
  float* wide;           // (slices, m, n) float32
  const float* add;      // (m, n) float32 added to an unsplit result, or nullptr
  const int* flags;      // dw: see xent_dz; a flagged stage's rows of x without a target are taken as zeros
  const int* targets;
  const float* scale;    // float16: see xent_scale
  int64_t rows, vocab;
};

// 4 columns of a result's row; columns past the width are padding and not stored. DX: zeros for a row without a target, which
// is asked for only where a total is not finite.
template <typename T, bool DX>
__device__ __forceinline__ void store4(const Products& s, int64_t row, int64_t col, f32x4 v) {
  if (col >= s.width) return;
  if (IS_F16<T>) v *= s.scale[1];
  if (DX) {
    const f32x4 odd = v * 0.f;
    if (odd[0] + odd[1] + odd[2] + odd[3] != 0.f) {
      const int t = s.targets[row];
      if (t < 0 || t >= s.vocab) v = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  if (s.out_f32) {
    float* o = (float*)s.out + row * s.width + col;
    if (s.vec) {
      *(f32x4*)o = v;
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (col + e < s.width) o[e] = v[e];
    return;
  }
  u16* o = (u16*)s.out + row * s.width + col;
  if (s.vec) {
    *(uint2*)o = make_uint2(T::pack2(v[0], v[1]), T::pack2(v[2], v[3]));
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (col + e < s.width) o[e] = T::pack(v[e]);
}

template <typename T, int BM, int PARTS, bool A_K>
__global__ __launch_bounds__(64 * Tile<BM>::WAVES, 2) void xent_product(Products s) {
#if defined(__HIP_DEVICE_COMPILE__)
  LIMN_XENT_LDS(BM)
  const int64_t tiles_m = (s.m + BM - 1) / BM, tiles_n = (s.n + BM - 1) / BM;
  int64_t tm, tn, slice;
  tile_of(tiles_m, tiles_n, tm, tn, slice);
  const int64_t m0 = tm * BM, n0 = tn * BM, k_lo = slice * s.chunk, k_hi = k_lo + s.chunk < s.k ? k_lo + s.chunk : s.k;
  const DmaOperand<BM, A_K, L::WAVES> da(s.a, s.a_rows, s.a_depth, s.a_stride, m0, k_lo, wave, lane);
  const DmaOperand<BM, false, L::WAVES> db(s.b, s.b_cols, s.b_depth, s.b_stride, n0, k_lo, wave, lane);
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
  tile_product<T, BM, PARTS, A_K, false, false>(da, db, s.part_a, s.part_b, A0, A1, B0, B1, (int)((k_hi - k_lo + BK - 1) / BK), 0, wave, lane, acc, fix);

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
          store4<T, A_K>(s, row, col, v);
        else
          *(f32x4*)(s.wide + (slice * s.m + row) * s.n + col) = v;
      }
    }
  }
#endif
}

// out = round(add + slices), or the same kept in float32 (s.wide). A workgroup is 64 threads of 4 elements by G runs
// of the slices, which are joined in order in LDS.
template <typename T, bool DX>
__global__ __launch_bounds__(1024) void xent_fold(Products s, const float* __restrict__ slices, int64_t count) {
  __shared__ f32x4 part[16][64];
  const int x = threadIdx.x, y = threadIdx.y, runs = blockDim.y;
  const int64_t total = s.m * s.n, i = (blockIdx.x * (int64_t)64 + x) * 4, run = (count + runs - 1) / runs;
  const int64_t k1 = (y + 1) * run < count ? (y + 1) * run : count;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (i < total) {
#pragma unroll 4
    for (int64_t k = y * run; k < k1; k++) v += *(const f32x4*)(slices + k * total + i);
  }
  part[y][x] = v;
  __syncthreads();
  if (y != 0 || i >= total) return;
  for (int g = 1; g < runs; g++) v += part[g][x];
  if (s.add != nullptr) v += *(const f32x4*)(s.add + i);
  if (s.out != nullptr) {
    const int64_t row = i / s.n;
    store4<T, DX>(s, row, i - row * s.n, v);
  } else {
    *(f32x4*)(s.wide + i) = v;
  }
}

// A matrix of `rows` rows of `width` elements and where its PARTS matrices of rows of `padded` elements go, `part` elements
// behind one another.
struct Copied {
  const void* src;
  u16* dst;
  int64_t rows, part;
};

// Two such matrices in one launch, zeros past the width: 8 consecutive elements a thread.
template <typename S, typename T, int PARTS>
__global__ __launch_bounds__(256) void xent_parts(Copied m0, Copied m1, int width, int padded) {
  const int chunks = padded / 8;
  const int64_t total = (m0.rows + m1.rows) * chunks;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t both = i / chunks;
    const int c = (int)(i - both * chunks) * 8;
    const bool second = both >= m0.rows;
    const int64_t row = second ? both - m0.rows : both, part = second ? m1.part : m0.part;
    const typename S::Storage* src = (const typename S::Storage*)(second ? m1.src : m0.src);
    u16* dst = second ? m1.dst : m0.dst;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = c + e < width ? S::load(src, row * width + c + e) : 0.f;
#pragma unroll
    for (int p = 0; p < PARTS; p++) {
      u16x8 w;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        u16 h = T::pack(v[e]);
        if (PARTS > 1) {
          const bool huge = !(fabsf(T::unpack(h)) <= 3.402823466e38f);
          // the largest numbers round past bfloat16's: cut off instead; an infinity or a NaN is its first part alone
          if (huge && fabsf(v[e]) <= 3.402823466e38f) h = (u16)(__float_as_uint(v[e]) >> 16);
          v[e] = fabsf(v[e]) <= 3.402823466e38f ? v[e] - T::unpack(h) : 0.f;
        }
        w[e] = h;
      }
      *(u16x8*)(dst + p * part + row * padded + c) = w;
    }
  }
}

// ---- plans ------------------------------------------------------------------------------------------------

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

constexpr int64_t FILL = 256;  // workgroups that give every CU one

int tile_for(int64_t m, int64_t n) { return ((m + 255) / 256) * ((n + 255) / 256) >= FILL ? 256 : 128; }

bool f32(const XentArgs& a) { return a.dtype == LIMN_HIP_FLOAT32; }
int parts_of(const XentArgs& a) { return f32(a) ? 3 : 1; }
int64_t padded_width(const XentArgs& a) { return up(a.width, 8); }

// Whether x and w go as they are: half widths in 16-byte rows.
bool rows16(const XentArgs& a) { return !f32(a) && a.width % 8 == 0; }
bool as_is(const XentArgs& a) { return rows16(a) && ((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0; }

// Rounds of tiles that keep the GPU: whole ones, or the part of one that smaller tiles or slices make of a few.
double rounds(int64_t tiles) { return tiles * 4 >= 3 * FILL ? (double)((tiles + FILL - 1) / FILL) : 1.3 * (double)tiles / FILL; }

// Vocabulary entries that go by at a time, a multiple of 256 and 1024 at least: what 32-bit offsets reach, dz
// within PIECE_BYTES or half as much again, and the copies of the weight's rows, where there are any, too. Of such sizes
// a backward takes the one whose dz and dw tiles leave the fewest CUs idle over all pieces, in units of one tile's stage of
// 64 deep; 16 of them are what a piece's launches and its tiles' beginnings and ends cost (4001 rows, width 760,
// vocabulary 50257: 3 pieces of 16384 and one of 1105, forward and backward, 1679 us; 2 of 20480 and one of 9297 1640).
int64_t piece_of(const XentArgs& a, bool backward, bool copies) {
  const int64_t whole = up(a.vocab, 256), half = PIECE_BYTES / 2 / parts_of(a), rows = (a.rows + 255) / 256, cols = (padded_width(a) + 255) / 256;
  const int64_t reach = (int64_t)0x70000000 / 2 / padded_width(a);
  int64_t most = reach;
  if (copies && half / padded_width(a) < most) most = half / padded_width(a);
  const int64_t fit = backward && half / (256 * rows) < most ? half / (256 * rows) : most;
  int64_t best = fit < 1024 ? 1024 : fit / 256 * 256;
  if (best >= whole) return whole;
  if (!backward) return best;
  double least = 0;
  const int64_t end = best + best / 2 < most ? best + best / 2 : most;
  for (int64_t p = up(best / 2 < 1024 ? 1024 : best / 2, 256), at = 0; p <= end; p += 256) {
    const int64_t pieces = (a.vocab + p - 1) / p, rest = a.vocab - (pieces - 1) * p;
    auto cost = [&](int64_t n) {
      const int64_t tiles = (n + 255) / 256;
      return rounds(rows * tiles) * (double)(a.width + 63) / 64 + rounds(tiles * cols) * (double)(a.rows + 63) / 64 + 16;
    };
    const double c = (double)(pieces - 1) * cost(p) + cost(rest);
    if (at++ == 0 || c < least) {
      least = c;
      best = p;
    }
  }
  return best < whole ? best : whole;
}

struct Cut {
  int tile;
  int64_t split, chunk;
};
// Tiles of 256 in as many slices of k as leave no more than a quarter of the CUs idle, where slices are long enough for
// their partial results; else as matmul.hip cuts its products. In three parts a slice is six times the work.
Cut cut(int64_t m, int64_t n, int64_t k, int parts) {
  const int64_t tiles = ((m + 255) / 256) * ((n + 255) / 256), work = parts == 3 ? 6 : 1;
  if (tiles < FILL && m > 128) {
    const int64_t split = FILL / tiles, chunk = up((k + split - 1) / split, BK);
    if (split * tiles * 4 >= 3 * FILL && (split == 1 || chunk * work >= 1024)) return {256, (k + chunk - 1) / chunk, chunk};
  }
  const MatmulPlan p = plan_matmul(MatmulShape{1, m, n, k * work});
  const int64_t chunk = up((k + p.split - 1) / p.split, BK);
  return {p.tile, (k + chunk - 1) / chunk, chunk};
}

int64_t product_bytes(int64_t m, int64_t n, int64_t k, int parts) {
  const Cut c = cut(m, n, k, parts);
  return c.split > 1 ? c.split * m * n * 4 : 0;
}

struct BwdPlan {
  int64_t piece, pieces, rows_pad, slices;  // slices: float32 (slices x result) bytes the products need at most
};

BwdPlan bwd_plan(const XentArgs& a, bool copies) {
  BwdPlan p;
  const int64_t width = padded_width(a);
  p.piece = piece_of(a, true, copies);
  p.pieces = (a.vocab + p.piece - 1) / p.piece;
  p.rows_pad = up(a.rows, 256);
  p.slices = 0;
  for (const int64_t n : {p.piece < a.vocab ? p.piece : a.vocab, a.vocab - (p.pieces - 1) * p.piece}) {
    const int64_t dx = product_bytes(a.rows, width, up(n, 64), parts_of(a)), dw = product_bytes(n, width, up(a.rows, 64), parts_of(a));
    if (dx > p.slices) p.slices = dx;
    if (dw > p.slices) p.slices = dw;
  }
  return p;
}

template <typename T, int BM, int PARTS>
int launch_stats(const Logits& l, hipStream_t stream) {
  const int64_t blocks = ((l.rows + BM - 1) / BM) * ((l.piece + BM - 1) / BM);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "xent: %lld workgroups exceed one launch", (long long)blocks);
  const dim3 grid((unsigned)blocks), block(64 * Tile<BM>::WAVES);
  if (l.width % BK == 0)
    hipLaunchKernelGGL((xent_stats<T, BM, PARTS, false>), grid, block, 0, stream, l);
  else
    hipLaunchKernelGGL((xent_stats<T, BM, PARTS, true>), grid, block, 0, stream, l);
  return check_hip(hipGetLastError(), "launching the cross entropy's logits");
}

template <typename T, int BM, int PARTS>
int launch_dz(const Logits& l, hipStream_t stream) {
  const int64_t blocks = ((l.rows + BM - 1) / BM) * (l.ldz / BM);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "xent: %lld workgroups exceed one launch", (long long)blocks);
  const dim3 grid((unsigned)blocks), block(64 * Tile<BM>::WAVES);
  if (l.width % BK == 0)
    hipLaunchKernelGGL((xent_dz<T, BM, PARTS, false>), grid, block, 0, stream, l);
  else
    hipLaunchKernelGGL((xent_dz<T, BM, PARTS, true>), grid, block, 0, stream, l);
  return check_hip(hipGetLastError(), "launching the cross entropy's gradient");
}

template <typename T, int PARTS, bool A_K>
int launch_product(Products s, const Cut& c, float* slices, float* acc, bool first, void* out, hipStream_t stream) {
  // unsplit: straight to out (the last piece of dx, or dw), or into the float32 totals; split: slices, then a fold
  const bool split = c.split > 1;
  const float* add = first ? nullptr : acc;
  s.chunk = c.chunk;
  s.out = split ? nullptr : out;
  s.wide = split ? slices : acc;
  s.add = split ? nullptr : add;
  const int64_t blocks = c.split * ((s.m + c.tile - 1) / c.tile) * ((s.n + c.tile - 1) / c.tile);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "xent: %lld workgroups exceed one launch", (long long)blocks);
  if (c.tile == 256)
    hipLaunchKernelGGL((xent_product<T, 256, PARTS, A_K>), dim3((unsigned)blocks), dim3(512), 0, stream, s);
  else
    hipLaunchKernelGGL((xent_product<T, 128, PARTS, A_K>), dim3((unsigned)blocks), dim3(256), 0, stream, s);
  const int rc = check_hip(hipGetLastError(), "launching a product of the cross entropy's gradient");
  if (rc != LIMN_HIP_OK || !split) return rc;
  s.out = out;
  s.wide = acc;
  s.add = add;
  // two loads a thread or more: a run's chain is what a small result waits for (48 x 512 of 62 slices: 18 -> 5 us)
  const int64_t groups = (s.m * s.n / 4 + 63) / 64;
  if (groups > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "xent: %lld workgroups exceed one launch", (long long)groups);
  const int runs = c.split < 8 ? 4 : c.split < 32 ? 8 : 16;
  hipLaunchKernelGGL((xent_fold<T, A_K>), dim3((unsigned)groups), dim3(64, runs), 0, stream, s, slices, c.split);
  return check_hip(hipGetLastError(), "launching the fold of a product's slices");
}

template <typename S, typename T, int PARTS>
int launch_parts(const Copied& m0, const Copied& m1, const XentArgs& a) {
  const int64_t padded = padded_width(a), groups = ((m0.rows + m1.rows) * (padded / 8) + 255) / 256;
  hipLaunchKernelGGL((xent_parts<S, T, PARTS>), dim3((unsigned)(groups < 16384 ? groups : 16384)), dim3(256), 0, a.stream, m0, m1, (int)a.width, (int)padded);
  return check_hip(hipGetLastError(), "launching an operand's parts");
}

// S: the operands' type, T: the type the products take, in PARTS parts.
template <typename S, typename T, int PARTS>
int fwd(const XentArgs& a) {
  const bool copies = !as_is(a);
  const int64_t piece = piece_of(a, false, copies), width = padded_width(a);
  const int bm = tile_for(a.rows, a.vocab);
  XentSpace space(a.workspace);
  const int64_t tiles = (a.vocab + bm - 1) / bm;
  Logits l = {};
  l.x = (const u16*)a.x, l.targets = a.targets, l.rows = a.rows, l.width = width, l.vocab = a.vocab;
  l.stats = (float2*)space.take(tiles * a.rows * 8);
  l.picked = (float*)space.take(a.rows * 4);
  u16* wp = nullptr;
  int rc = LIMN_HIP_OK;
  if (copies) {
    u16* xp = (u16*)space.take(PARTS * a.rows * width * 2);
    wp = (u16*)space.take(PARTS * piece * width * 2);
    l.x = xp;
    l.part_x = a.rows * width;
  }
  for (int64_t v0 = 0; v0 < a.vocab && rc == LIMN_HIP_OK; v0 += piece) {
    const typename S::Storage* w = (const typename S::Storage*)a.w + v0 * a.width;
    l.v0 = v0;
    l.piece = a.vocab - v0 < piece ? a.vocab - v0 : piece;
    l.tile0 = v0 / bm;
    l.w = (const u16*)w;
    if (copies) {
      l.w = wp;
      l.part_w = l.piece * width;
      const Copied rows = {a.x, (u16*)l.x, v0 == 0 ? a.rows : 0, l.part_x};
      if ((rc = launch_parts<S, T, PARTS>(rows, Copied{w, wp, l.piece, l.part_w}, a)) != LIMN_HIP_OK) return rc;
    }
    rc = bm == 256 ? launch_stats<T, 256, PARTS>(l, a.stream) : launch_stats<T, 128, PARTS>(l, a.stream);
  }
  if (rc != LIMN_HIP_OK) return rc;
  if (a.rows >= 32 * FILL)
    hipLaunchKernelGGL((xent_rows<32>), dim3((unsigned)((a.rows + 31) / 32)), dim3(256), 0, a.stream, l.stats, l.picked, a.targets, (float*)a.o0, (float*)a.o1, a.rows,
                       tiles, a.vocab);
  else
    hipLaunchKernelGGL((xent_rows<4>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, a.stream, l.stats, l.picked, a.targets, (float*)a.o0, (float*)a.o1, a.rows,
                       tiles, a.vocab);
  return check_hip(hipGetLastError(), "launching the cross entropy's rows");
}

template <typename S, typename T, int PARTS>
int bwd(const XentArgs& a) {
  const bool copies = !as_is(a);
  const BwdPlan p = bwd_plan(a, copies);
  const int64_t width = padded_width(a);
  XentSpace space(a.workspace);
  Logits l = {};
  l.x = (const u16*)a.x, l.targets = a.targets, l.rows = a.rows, l.width = width, l.vocab = a.vocab, l.lse = a.lse_in, l.g = a.g;
  l.dz = (u16*)space.take(PARTS * p.rows_pad * p.piece * 2);
  l.flags = (int*)space.take(p.rows_pad / 64 * 4);
  if (IS_F16<T>) {
    float* scale = (float*)space.take(8);
    hipLaunchKernelGGL(xent_scale, dim3(1), dim3(1024), 0, a.stream, a.g, a.targets, a.rows, a.vocab, scale);
    if (const int bad = check_hip(hipGetLastError(), "launching the gradient's scale"); bad != LIMN_HIP_OK) return bad;
    l.scale = scale;
  }
  float* slices = (float*)space.take(p.slices);
  float* acc = p.pieces > 1 ? (float*)space.take(a.rows * width * 4) : nullptr;
  u16* wp = nullptr;
  int rc = LIMN_HIP_OK;
  if (copies) {
    u16* xp = (u16*)space.take(PARTS * a.rows * width * 2);
    wp = (u16*)space.take(PARTS * p.piece * width * 2);
    l.x = xp;
    l.part_x = a.rows * width;
  }
  for (int64_t v0 = 0; v0 < a.vocab; v0 += p.piece) {
    const bool first = v0 == 0, last = v0 + p.piece >= a.vocab;
    const typename S::Storage* w = (const typename S::Storage*)a.w + v0 * a.width;
    l.v0 = v0;
    l.piece = last ? a.vocab - v0 : p.piece;
    l.ldz = up(l.piece, 256);
    l.part_dz = p.rows_pad * l.ldz;
    l.w = (const u16*)w;
    if (copies) {
      l.w = wp;
      l.part_w = l.piece * width;
      const Copied rows = {a.x, (u16*)l.x, v0 == 0 ? a.rows : 0, l.part_x};
      if ((rc = launch_parts<S, T, PARTS>(rows, Copied{w, wp, l.piece, l.part_w}, a)) != LIMN_HIP_OK) return rc;
    }
    rc = tile_for(a.rows, l.ldz) == 256 ? launch_dz<T, 256, PARTS>(l, a.stream) : launch_dz<T, 128, PARTS>(l, a.stream);
    if (rc != LIMN_HIP_OK) return rc;
    Products s = {};
    s.rows = a.rows, s.vocab = a.vocab, s.targets = a.targets, s.flags = l.flags, s.scale = l.scale;
    s.out_f32 = f32(a), s.width = a.width, s.n = width;
    s.a = l.dz, s.part_a = l.part_dz, s.b = l.w, s.part_b = l.part_w, s.m = a.rows, s.k = up(l.piece, 64);
    s.a_rows = p.rows_pad, s.a_depth = l.ldz, s.a_stride = l.ldz, s.b_depth = l.piece, s.b_stride = width, s.b_cols = width;
    s.vec = a.width % 4 == 0 && (uintptr_t)a.o0 % (f32(a) ? 16 : 8) == 0;
    rc = launch_product<T, PARTS, true>(s, cut(s.m, s.n, s.k, PARTS), slices, acc, first, last ? a.o0 : nullptr, a.stream);
    if (rc != LIMN_HIP_OK) return rc;
    s.b = l.x, s.part_b = l.part_x, s.m = l.piece, s.k = up(a.rows, 64);
    s.a_rows = l.ldz, s.a_depth = p.rows_pad, s.b_depth = a.rows;
    void* dw = (typename S::Storage*)a.o1 + v0 * a.width;
    s.vec = a.width % 4 == 0 && (uintptr_t)dw % (f32(a) ? 16 : 8) == 0;
    rc = launch_product<T, PARTS, false>(s, cut(s.m, s.n, s.k, PARTS), slices, nullptr, true, dw, a.stream);
    if (rc != LIMN_HIP_OK) return rc;
  }
  return LIMN_HIP_OK;
}

}  // namespace

// every operand's bytes within 32-bit offsets of a base (a tile may reach 256 rows past its end)
bool xent_sizes_ok(const XentArgs& a) {
  const int64_t most = (int64_t)0x7f000000 / 2, width = padded_width(a), piece = piece_of(a, true, false), ahead = piece_of(a, false, false);
  return (a.rows + 512) * width < most && (ahead + 512) * width < most && (up(a.rows, 256) + 512) * piece < most && (piece + 512) * width < most;
}

namespace {

int64_t workspace_of(const XentArgs& a, bool backward, bool copies) {
  const int64_t width = padded_width(a), parts = parts_of(a), row = parts * 2 * width;
  int64_t need = copies ? xent_align(a.rows * row) + xent_align(piece_of(a, backward, copies) * row) : 0;
  if (!backward) return need + xent_align(((a.vocab + 127) / 128) * a.rows * 8) + xent_align(a.rows * 4);
  const BwdPlan p = bwd_plan(a, copies);
  need += xent_align(parts * p.rows_pad * p.piece * 2) + xent_align(p.rows_pad / 64 * 4) + xent_align(8) + xent_align(p.slices);
  return need + (p.pieces > 1 ? xent_align(a.rows * width * 4) : 0);
}

}  // namespace

// Enough whether or not the call's buffers are aligned as their sizes allow.
int64_t xent_workspace(const XentArgs& a, bool backward) {
  const int64_t copied = workspace_of(a, backward, true), plain = rows16(a) ? workspace_of(a, backward, false) : 0;
  return copied > plain ? copied : plain;
}

int launch_xent_fwd(const XentArgs& a) {
  if (f32(a)) return fwd<F32, BF16, 3>(a);
  return a.dtype == LIMN_HIP_BFLOAT16 ? fwd<BF16, BF16, 1>(a) : fwd<F16, F16, 1>(a);
}
int launch_xent_bwd(const XentArgs& a) {
  if (f32(a)) return bwd<F32, BF16, 3>(a);
  return a.dtype == LIMN_HIP_BFLOAT16 ? bwd<BF16, BF16, 1>(a) : bwd<F16, F16, 1>(a);
}

}  // namespace limn
