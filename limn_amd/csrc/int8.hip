// A linear layer in 8-bit integers (include/limn_hip.h, limn_hip_int8_linear) and the bringing of rows to 8 bits
// (limn_hip_quantize_rows):
//
//   s = max(max |x| / 127, 2^-126),  x8 = round(x / s) (ties to even),  y = (x8 . w8) s scale + bias.
//
// Sums of products are whole numbers in 32 bits, exact up to 2^17 terms of 127 * 128, so any order of adding gives the same.
// Rows of x8 are padded with zeros to whole multiples of 256 bytes: what a stage holds of a weight's next row is multiplied by 0, and
// rows past an operand's end read as zeros, so the loops have no tests of bounds.
//
// int8_tiles (many rows; bound by the matrix cores): output tiles of 256 x 256, 128 x 128 or 64 x 64 on 4 waves, one a SIMD, each
// with a quarter as accumulators of v_mfma_i32_32x32x32_i8. A wave's 128 x 128 takes 8 reads of LDS for 16 products, half
// of what 8 waves of 128 x 64 do, whose LDS was busy all the time. Stages of 64 bytes a row (128 in the smaller tiles) go straight to LDS
// (buffer_load ... lds) into one of four buffers, three stages ahead. Operands are read a k
// step ahead, the last one's of a stage in the next stage, which has landed by then.
//
// int8_few (up to 16 rows; bound by reading the weight once): a wave has 16 outputs and a part of the width, its bytes read from
// memory straight into operands of v_mfma_i32_16x16x64_i8; the waves of a workgroup add their sums in LDS. A few inputs are brought
// to 8 bits by every workgroup, while its weights are on their way.

#include "common.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace limn {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int PAD = 256;     // rows of x8 are padded to whole multiples of this: four stages

// the s_waitcnt immediate that leaves the newest n vector memory operations in flight, and the other counters free
constexpr int wait_vm(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); }

struct Int8Args {
  const void* x;
  const void* w;
  const float* w_scales;
  const void* bias;  // of x's type, or nullptr
  void* out;
  int dtype;
  int64_t rows, width, outputs, out_row;  // out_row: outputs between rows of out, more than `outputs` where a call goes in slabs
  void* workspace;
  hipStream_t stream;
  int64_t padded() const { return (width + PAD - 1) / PAD * PAD; }
};

constexpr int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The copy of the weight with aligned rows that a call needs where its rows are not.
bool needs_copy(const void* w, int64_t width) { return width % 16 != 0 || (uintptr_t)w % 16 != 0; }

// Outputs that there is room to copy at a time. Of a width whose rows may be aligned a whole weight may not be spared for a start that
// is not: such a call goes in slabs of some 64 MB, whole tiles each (300 x 4096 x 50000, four of them: 259 us, 240 in one; slabs of 16 MB
// 331).
int64_t copied_outputs(int64_t width, int64_t outputs) {
  if (width % 16 != 0) return outputs;
  const int64_t padded = (width + PAD - 1) / PAD * PAD, slab = std::max<int64_t>(((int64_t)1 << 26) / padded / 256, 1) * 256;
  return std::min(outputs, slab);
}

// 8 consecutive elements
template <typename T>
struct Eight {
  u16x8 x;
  __device__ __forceinline__ void load(const u16* p) { x = *(const u16x8*)p; }
  __device__ __forceinline__ float at(int i) const { return T::unpack(x[i]); }
};
template <>
struct Eight<F32> {
  f32x4 lo, hi;
  __device__ __forceinline__ void load(const float* p) {
    lo = *(const f32x4*)p;
    hi = *(const f32x4*)(p + 4);
  }
  __device__ __forceinline__ float at(int i) const { return i < 4 ? lo[i & 3] : hi[i & 3]; }
};

// A row's scale, from its largest magnitude (an infinity where the row has one or a NaN), and its numbers.
struct Rounding {
  float s;
  bool fine;
  __device__ __forceinline__ explicit Rounding(float top) : s(fmaxf(top / 127.f, 0x1p-126f)), fine(top < __builtin_inff()) {}
  __device__ __forceinline__ float scale() const { return fine ? s : __builtin_nanf(""); }
  __device__ __forceinline__ int operator()(float v) const { return fine ? (int)rintf(v / s) : 0; }
  template <typename E>
  __device__ __forceinline__ uint2 eight(const E& x) const {
    unsigned lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      lo |= ((unsigned)(*this)(x.at(i)) & 255u) << (8 * i);
      hi |= ((unsigned)(*this)(x.at(4 + i)) & 255u) << (8 * i);
    }
    return make_uint2(lo, hi);
  }
};

constexpr int HELD = 4;  // eights a thread of quantize_rows holds between its two uses: 8192 elements a row

// A workgroup a row: its largest magnitude, then its numbers, `stride` bytes a row, zeros behind the width. A row with an
// infinity or a NaN gets the scale NaN and zeros. With `vec` (rows of whole aligned eights) the row's first 8192 elements are read
// once. Workgroups past the rows copy a weight's rows, `width` bytes, to w_out with zeros behind, four bytes a thread from wherever they
// begin (16 x 4097 x 8192 29 us, byte by byte 54).
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows(const typename T::Storage* __restrict__ x, signed char* __restrict__ out, float* __restrict__ scales, int64_t rows, int64_t width,
                                                     int64_t stride, int vec, const signed char* __restrict__ w, signed char* __restrict__ w_out, int64_t outputs) {
  __shared__ float tops[4];
  if (blockIdx.x >= rows) {
    for (int64_t r = blockIdx.x - rows; r < outputs; r += gridDim.x - rows)
      for (int64_t i = threadIdx.x * 4; i < stride; i += 1024) {
        unsigned x = 0;
        if (i + 4 <= width) {
          __builtin_memcpy(&x, w + r * width + i, 4);
        } else {
          for (int b = 0; b < 4 && i + b < width; b++) x |= (unsigned)(unsigned char)w[r * width + i + b] << (8 * b);
        }
        *(unsigned*)(w_out + r * stride + i) = x;
      }
    return;
  }
  const typename T::Storage* row = x + blockIdx.x * width;
  signed char* o = out + blockIdx.x * stride;
  float top = 0.f, odd = 0.f;
  Eight<T> held[HELD];
  auto look = [&](float v) __attribute__((always_inline)) {
    top = fmaxf(top, fabsf(v));
    odd = fmaf(v, 0.f, odd);  // NaN once an infinity or a NaN was there
  };
  const int64_t eights = vec ? width / 8 : 0;
#pragma unroll
  for (int h = 0; h < HELD; h++)
    if (h * 256 + threadIdx.x < eights) held[h].load(row + (h * 256 + threadIdx.x) * 8);
#pragma unroll
  for (int h = 0; h < HELD; h++)
    if (h * 256 + threadIdx.x < eights) {
#pragma unroll
      for (int i = 0; i < 8; i++) look(held[h].at(i));
    }
  for (int64_t i = (vec ? HELD * 2048 : 0) + threadIdx.x; i < width; i += 256) look(T::load(row, i));
  if (odd != odd) top = __builtin_inff();
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const Rounding by(top);
  if (threadIdx.x == 0) scales[blockIdx.x] = by.scale();
#pragma unroll
  for (int h = 0; h < HELD; h++)
    if (h * 256 + threadIdx.x < eights) *(uint2*)(o + (h * 256 + threadIdx.x) * 8) = by.eight(held[h]);
  for (int64_t i = (vec ? HELD * 2048 : 0) + threadIdx.x; i < width; i += 256) o[i] = (signed char)by(T::load(row, i));
  for (int64_t i = width + threadIdx.x; i < stride; i += 256) o[i] = 0;
}

// One operand's tile of ROWS rows from row0 on: the copy of a stage to LDS, and the matrix instruction's operands.
// STAGE bytes a row; chunk c of LDS row r lies at c ^ swizzle(r), so that the 16 rows a read serves in a cycle (those of one parity
// of r >> 2 in 32) are in 16 places of the 64 banks.
template <int ROWS, int STAGE>
struct Tile {
  static constexpr int BYTES = ROWS * STAGE, PASSES = BYTES / (1024 * 4), CHUNKS = STAGE / 16, RPI = 64 / CHUNKS, KK = STAGE / 32;
  static __device__ __forceinline__ int swizzle(int r) { return STAGE == 64 ? (r >> 3) & 3 : (r >> 1) & 7; }
  const char* base;
  int64_t extent;  // bytes from base to the operand's end
  int voff[PASSES];
  __device__ __forceinline__ Tile(const signed char* p, int64_t rows, int64_t stride, int64_t row0, int wave, int lane) {
    base = (const char*)p + row0 * stride;
    extent = (rows - row0) * stride;
#pragma unroll
    for (int q = 0; q < PASSES; q++) {
      const int r = (q * 4 + wave) * RPI + lane / CHUNKS;
      voff[q] = (int)(r * stride) + ((lane % CHUNKS) ^ swizzle(r)) * 16;
    }
  }
  __device__ __forceinline__ void copy(char* tile, int stage, int wave) const {
    const int64_t off = (int64_t)stage * STAGE, left = extent - off;
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)(base + off), (short)0, (int)(left < 0 ? 0 : left < 0x7fffffff ? left : 0x7fffffff), 0x00020000);
#pragma unroll
    for (int q = 0; q < PASSES; q++) __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(tile + (q * 4 + wave) * 1024), 16, voff[q], 0, 0, 0);
  }
  // lane l: bytes 32 kk + 16 (l / 32) .. + 15 of row row0 + l % 32; kk a place in rd
  static __device__ __forceinline__ void offsets(int row0, int lane, int* rd) {
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int kk = 0; kk < KK; kk++) rd[kk] = (row0 + r) * STAGE + ((2 * kk + h) ^ swizzle(r)) * 16;
  }
  static __device__ __forceinline__ i32x4 operand(const char* tile, int at, int t) { return *(const i32x4*)(tile + at + t * 32 * STAGE); }
};

// A sum times the weight's scale, then times the scale of x, which may be as large as x, and the bias or 0. Every kernel gives the
// same bits: one operation by name, and a float32 before it is rounded to float16 (an instruction that does both rounds but once).
__device__ __forceinline__ float scaled(int sum, float w_scale, float x_scale, float bias) {
  float y = fmaf((float)sum * w_scale, x_scale, bias);
  asm("" : "+v"(y));
  return y;
}

template <typename T, int BM, int STAGE>
__global__ __launch_bounds__(256, BM * STAGE > 8192 ? 1 : 2) void int8_tiles(const signed char* __restrict__ x8, const float* __restrict__ scales, const signed char* __restrict__ w8,
                                                                    int64_t w_stride, Int8Args a) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr int WT = BM / 2, TM = WT / 32;  // a wave's tile, WT x WT
  typedef Tile<BM, STAGE> O;
  constexpr int FLIGHT = 2 * O::PASSES, KK = O::KK;  // copies of a stage and wave; k steps of a stage
  __shared__ __attribute__((aligned(1024))) char A0[O::BYTES], A1[O::BYTES], A2[O::BYTES], A3[O::BYTES];
  __shared__ __attribute__((aligned(1024))) char B0[O::BYTES], B1[O::BYTES], B2[O::BYTES], B3[O::BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n32 = lane & 31;
  const int wm = wave >> 1, wn = wave & 1;
  const int64_t tiles_n = (a.outputs + BM - 1) / BM, tiles_m = (a.rows + BM - 1) / BM;
  int64_t id = blockIdx.x;
  if (gridDim.x % 8 == 0) id = (id % 8) * (gridDim.x / 8) + id / 8;  // an XCD's workgroups: a run of tiles, 4 tile rows at a time
  constexpr int64_t GROUP = 4;
  const int64_t group = id / (GROUP * tiles_n), first = group * GROUP, live = tiles_m - first < GROUP ? tiles_m - first : GROUP;
  const int64_t m0 = (first + (id - group * GROUP * tiles_n) % live) * BM, n0 = (id - group * GROUP * tiles_n) / live * BM;
  const int64_t padded = (a.width + PAD - 1) / PAD * PAD;
  // the largest tiles take whole fours of stages: a way out between them cost the accumulators' way through memory
  const int stages = (int)(BM == 256 ? padded / STAGE : (a.width + STAGE - 1) / STAGE);

  i32x16 acc[TM][TM];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TM; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
  const O da(x8, a.rows, padded, m0, wave, lane), db(w8, a.outputs, w_stride, n0, wave, lane);
  int rda[KK], rdb[KK];
  O::offsets(wm * WT, lane, rda);
  O::offsets(wn * WT, lane, rdb);
  i32x4 av[2][TM], bv[2][TM];
  auto read = [&](const char* at, const char* bt, int kk, i32x4* ao, i32x4* bo) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; i++) ao[i] = O::operand(at, rda[kk], i);
#pragma unroll
    for (int j = 0; j < TM; j++) bo[j] = O::operand(bt, rdb[kk], j);
  };
  auto multiply = [&](const i32x4* ao, const i32x4* bo) __attribute__((always_inline)) {
    // the weight's operand first: a lane then holds 4 consecutive outputs of a row
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TM; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bo[j], ao[i], acc[i][j], 0, 0, 0);
  };
  // stage st from (at, bt), whose first operands are in registers; (an, bn) the next one's, (af, bf) where stage st + 3 goes:
  // the buffer that every wave is done with at the barrier
  auto stage = [&](const char* at, const char* bt, const char* an, const char* bn, char* af, char* bf, int st) __attribute__((always_inline)) {
    // this wave's part of stage st + 1 has landed, st + 2 is on its way; then every wave's has
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(FLIGHT) : "memory");
    da.copy(af, st + 3, wave);
    db.copy(bf, st + 3, wave);
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
      if (kk + 1 < KK)
        read(at, bt, kk + 1, av[(kk + 1) & 1], bv[(kk + 1) & 1]);
      else
        read(an, bn, 0, av[0], bv[0]);
      multiply(av[kk & 1], bv[kk & 1]);
    }
    // the copies and the reads for the next k step among the products
#pragma unroll
    for (int k = 0; k < KK; k++)
#pragma unroll
      for (int r = 0; r < 2 * TM; r++) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if ((k * 2 * TM + r) % 2 == 0) __builtin_amdgcn_sched_group_barrier(0x020, FLIGHT / (KK * TM), 0);
        __builtin_amdgcn_sched_group_barrier(0x008, TM > 1 ? TM / 2 : 1, 0);
      }
  };
  da.copy(A0, 0, wave);
  db.copy(B0, 0, wave);
  da.copy(A1, 1, wave);
  db.copy(B1, 1, wave);
  da.copy(A2, 2, wave);
  db.copy(B2, 2, wave);
  __builtin_amdgcn_s_waitcnt(wait_vm(2 * FLIGHT));
  __syncthreads();
  read(A0, B0, 0, av[0], bv[0]);
  for (int st = 0; st < stages; st += 4) {
    stage(A0, B0, A1, B1, A3, B3, st);
    if (BM < 256 && st + 1 >= stages) break;
    stage(A1, B1, A2, B2, A0, B0, st + 1);
    if (BM < 256 && st + 2 >= stages) break;
    stage(A2, B2, A3, B3, A1, B1, st + 2);
    if (BM < 256 && st + 3 >= stages) break;
    stage(A3, B3, A0, B0, A2, B2, st + 3);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no copy may land in what is staged below
  __syncthreads();

  // Through LDS, so that a store instruction writes whole row segments: 32 rows of a wave's sums at a time, 16-byte chunk c of row r
  // at c ^ (r & 7). Coming back, a lane has 8 outputs of a row, the same ones for every row. Where rows of the result are not
  // aligned, 16-bit results go back to LDS and out in the aligned eights of their row, its first and last few one by one (1021 x 760 x 2279:
  // 17.7 us, 20.2 with one output a lane); float32 ones in turn.
  typedef typename T::Storage S;
  constexpr int LPR = WT / 8, RPI = 64 / LPR;  // lanes a row, rows at a time
  static_assert(32 * WT * 4 <= O::BYTES, "a wave's rows fit a buffer");
  char* const region = wave == 0 ? A0 : wave == 1 ? A1 : wave == 2 ? B0 : B1;
  S* out = (S*)a.out;
  const S* bias = (const S*)a.bias;
  const int64_t col = n0 + wn * WT + (lane % LPR) * 8;
  const bool wide = a.out_row % 8 == 0 && ((uintptr_t)out & 15) == 0;
  float ws[8], bs[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    ws[e] = col + e < a.outputs ? a.w_scales[col + e] : 0.f;
    bs[e] = bias != nullptr && col + e < a.outputs ? T::load(bias, col + e) : 0.f;
  }
  float xs[TM];  // the scales of the 32 rows, one a lane of each half
#pragma unroll
  for (int i = 0; i < TM; i++) xs[i] = scales[min(m0 + wm * WT + i * 32 + n32, a.rows - 1)];
#pragma unroll
  for (int i = 0; i < TM; i++) {
#pragma unroll
    for (int j = 0; j < TM; j++)
#pragma unroll
      for (int q = 0; q < 4; q++)
        *(i32x4*)(region + n32 * WT * 4 + ((8 * j + 2 * q + h) ^ (n32 & 7)) * 16) = i32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
    if (sizeof(S) == 4 && !wide) {
      constexpr int SPAN = WT < 64 ? WT : 64;
#pragma unroll 1
      for (int cs = 0; cs < WT / SPAN; cs++) {
        const int in = cs * 64 + lane % SPAN;
        const int64_t c = n0 + wn * WT + in;
        const float w = c < a.outputs ? a.w_scales[c] : 0.f, b = bias != nullptr && c < a.outputs ? T::load(bias, c) : 0.f;
#pragma unroll 4  // run once a block: its own fetch is most of its time if it is unrolled
        for (int r0 = 0; r0 < 32; r0 += 64 / SPAN) {
          const int r = r0 + lane / SPAN;
          const int64_t row = m0 + wm * WT + i * 32 + r;
          const float v = scaled(*(const int*)(region + r * WT * 4 + ((in >> 2) ^ (r & 7)) * 16 + (in & 3) * 4), w, __shfl(xs[i], r), b);
          if (row < a.rows && c < a.outputs) T::store(out, row * a.out_row + c, v);
        }
      }
      __builtin_amdgcn_wave_barrier();
      continue;
    }
#pragma unroll
    for (int it = 0; it < 32 / RPI; it++) {
      const int r = it * RPI + lane / LPR;
      const int64_t row = m0 + wm * WT + i * 32 + r;
      const float s = __shfl(xs[i], r);
      float y[8];
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const i32x4 c = *(const i32x4*)(region + r * WT * 4 + ((2 * (lane % LPR) + half) ^ (r & 7)) * 16);
#pragma unroll
        for (int e = 0; e < 4; e++) y[4 * half + e] = scaled(c[e], ws[4 * half + e], s, bs[4 * half + e]);
      }
      if constexpr (sizeof(S) == 2)
        if (!wide) {  // over the row's sums, which all of its lanes have read
          *(u32x4*)(region + r * WT * 4 + ((lane % LPR) ^ (r % LPR)) * 16) = u32x4{T::pack2(y[0], y[1]), T::pack2(y[2], y[3]), T::pack2(y[4], y[5]), T::pack2(y[6], y[7])};
          continue;
        }
      if (row >= a.rows || col >= a.outputs) continue;
      S* o = out + row * a.out_row + col;
      if constexpr (std::is_same<T, F32>::value) {
        *(f32x4*)o = f32x4{y[0], y[1], y[2], y[3]};
        *(f32x4*)(o + 4) = f32x4{y[4], y[5], y[6], y[7]};
      } else {
        *(u32x4*)o = u32x4{T::pack2(y[0], y[1]), T::pack2(y[2], y[3]), T::pack2(y[4], y[5]), T::pack2(y[6], y[7])};
      }
    }
    __builtin_amdgcn_wave_barrier();
    if constexpr (sizeof(S) == 2)
      if (!wide) {
        const int64_t c0 = n0 + wn * WT;
        const int many = (int)min((int64_t)WT, a.outputs - c0), j = lane % LPR;  // outputs of this wave; below 1: none
#pragma unroll 2
        for (int it = 0; it < 32 / RPI; it++) {
          const int r = it * RPI + lane / LPR;
          const int64_t row = m0 + wm * WT + i * 32 + r;
          const char* const from = region + r * WT * 4;
          auto word = [&](int w) __attribute__((always_inline)) { return *(const unsigned*)(from + (((w >> 2) & (LPR - 1)) ^ (r % LPR)) * 16 + (w & 3) * 4); };
          S* o = out + row * a.out_row + c0;
          const int before = (int)((16 - ((uintptr_t)o & 15)) & 15) / 2, at = before + 8 * j;  // the outputs before the first boundary
          unsigned w[5];
#pragma unroll
          for (int e = 0; e < 5; e++) w[e] = word((at >> 1) + e);  // past the row's end: its beginning, not used
          u32x4 x;
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = at & 1 ? (w[e] >> 16) | (w[e + 1] << 16) : w[e];
          if (row >= a.rows || many < 1) continue;
          if (at + 8 <= many) *(u32x4*)(o + at) = x;
          const int left = min(before, many), right = (many - left) % 8;
          for (int e = j; e < left; e += LPR) o[e] = (S)(word(e >> 1) >> (16 * (e & 1)));
          for (int e = many - right + j; e < many; e += LPR) o[e] = (S)(word(e >> 1) >> (16 * (e & 1)));
        }
        __builtin_amdgcn_wave_barrier();
      }
  }
#endif
}

// Inputs that every workgroup of int8_few brings to 8 bits for itself, in place of a launch before it: up to 8192 bytes for up to 1024
// workgroups. (By itself and by a launch: 1 x 4096 x 4096 8.9 and 11.8 us, 2 x 4096 x 8192 10.1 and 11.9, 16 x 512 x 2048 9.0 and 12.1; 4 x
// 4096 x 8192 14.0 and 11.9, 1 x 1024 x 50000 15.9 and 15.1, 4 x 1024 x 50000 19.7 and 16.2.)
constexpr int OWN_BYTES = 8192, OWN_OUTPUTS = 16384;
constexpr int OWN_ROW = 16;  // bytes between two rows, to part their banks

// 16 outputs of up to 16 rows; the width in pairs of 64 bytes, 4 of a wave's in flight while 4 are multiplied. OWN: x is not in 8 bits
// yet (rows of whole aligned eights, rows * padded at most OWN_BYTES).
template <typename T, bool OWN>
__global__ __launch_bounds__(256) void int8_few(const signed char* __restrict__ x8, const float* __restrict__ scales, const signed char* __restrict__ w8, int64_t w_stride, Int8Args a) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr int U = 4, STEP = 4 * U;  // pairs of a wave, and of the workgroup, in a batch
  __shared__ __attribute__((aligned(16))) int sums[4 * 256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int64_t n0 = blockIdx.x * (int64_t)16, padded = (a.width + PAD - 1) / PAD * PAD;
  const int pairs = (int)((a.width + 127) / 128);
  const int64_t left = (a.outputs - n0) * w_stride;
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)(w8 + n0 * w_stride), (short)0, (int)(left < 0x7fffffff ? left : 0x7fffffff), 0x00020000);
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)x8, (short)0, (int)(a.rows * padded), 0x00020000);
  const int wv = (int)(n * w_stride) + 16 * g, xv = (int)(n * padded) + 16 * g;
  __shared__ __attribute__((aligned(16))) signed char own[OWN ? OWN_BYTES + 16 * OWN_ROW : 16];
  __shared__ float own_scales[16], tops[4];
  i32x4 acc = {0, 0, 0, 0};
  struct Batch {
    i32x4 w[2 * U], x[2 * U];
  };
  auto load = [&](Batch& b, int p0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const int p = p0 + 4 * u, off = p * 128 + k * 64;  // past the width: zeros, and nothing of the next row is read
        b.w[2 * u + k] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, p < pairs ? wv + off : 0x7ffffff0, 0, 0));
        if (!OWN) b.x[2 * u + k] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rx, p < pairs ? xv + off : 0x7ffffff0, 0, 0));
      }
  };
  auto from_own = [&](Batch& b, int p0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const int p = p0 + 4 * u;
        b.x[2 * u + k] = p < pairs && n < a.rows ? *(const i32x4*)(own + n * (padded + OWN_ROW) + p * 128 + k * 64 + 16 * g) : i32x4{0, 0, 0, 0};
      }
  };
  auto multiply = [&](const Batch& b) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2 * U; u++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b.w[u], b.x[u], acc, 0, 0, 0);
  };
  Batch b0, b1;
  load(b0, wave);
  if constexpr (OWN) {  // as quantize_rows does, by one, two or four waves a row
    const int share = a.rows == 1 ? 4 : a.rows == 2 ? 2 : 1, at_once = 4 / share, eights = (int)(a.width / 8);
    for (int r0 = 0; r0 < a.rows; r0 += at_once) {
      const int r = r0 + wave / share, first = (wave % share) * 64 + lane;
      const typename T::Storage* row = (const typename T::Storage*)a.x + r * a.width;
      float top = 0.f, odd = 0.f;
      if (r < a.rows)
        for (int i = first; i < eights; i += share * 64) {
          Eight<T> x;
          x.load(row + i * 8);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            top = fmaxf(top, fabsf(x.at(e)));
            odd = fmaf(x.at(e), 0.f, odd);
          }
        }
      if (odd != odd) top = __builtin_inff();
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
      if (lane == 0) tops[wave] = top;
      __syncthreads();
      for (int w = 0; w < share; w++) top = fmaxf(top, tops[wave / share * share + w]);
      const Rounding by(top);
      if (r < a.rows) {
        if (first == 0) own_scales[r] = by.scale();
        for (int i = first; i < (int)(padded / 8); i += share * 64) {
          uint2 y = {0u, 0u};
          if (i < eights) {
            Eight<T> x;
            x.load(row + i * 8);
            y = by.eight(x);
          }
          *(uint2*)(own + r * (padded + OWN_ROW) + i * 8) = y;
        }
      }
      __syncthreads();
    }
  }
  for (int p = wave; p < pairs; p += 2 * STEP) {
    if (p + STEP < pairs) load(b1, p + STEP);
    if (OWN) from_own(b0, p);
    multiply(b0);
    if (p + STEP >= pairs) break;
    if (p + 2 * STEP < pairs) load(b0, p + 2 * STEP);
    if (OWN) from_own(b1, p + STEP);
    multiply(b1);
  }
  *(i32x4*)&sums[(wave * 16 + n) * 16 + 4 * g] = acc;  // row n, outputs 4 g .. + 3
  __syncthreads();
  typedef typename T::Storage S;
  const S* bias = (const S*)a.bias;
  const int i = threadIdx.x;
  const int sum = (sums[i] + sums[256 + i]) + (sums[512 + i] + sums[768 + i]);
  const int64_t row = i >> 4, col = n0 + (i & 15);
  if (row >= a.rows || col >= a.outputs) return;
  T::store((S*)a.out, row * a.out_row + col, scaled(sum, a.w_scales[col], OWN ? own_scales[row] : scales[row], bias != nullptr ? T::load(bias, col) : 0.f));
#endif
}

int64_t tiles(const Int8Args& a, int64_t m) { return ((a.rows + m - 1) / m) * ((a.outputs + m - 1) / m); }

template <typename T, int BM, int STAGE>
int tiles_of(const Int8Args& a, const signed char* x8, const float* scales, const signed char* w8, int64_t w_stride) {
  hipLaunchKernelGGL((int8_tiles<T, BM, STAGE>), dim3((unsigned)tiles(a, BM)), dim3(256), 0, a.stream, x8, scales, w8, w_stride, a);
  return check_hip(hipGetLastError(), "launching the 8-bit product");
}

template <typename T, bool OWN>
int few_of(const Int8Args& a, const signed char* x8, const float* scales, const signed char* w8, int64_t w_stride) {
  hipLaunchKernelGGL((int8_few<T, OWN>), dim3((unsigned)((a.outputs + 15) / 16)), dim3(256), 0, a.stream, x8, scales, w8, w_stride, a);
  return check_hip(hipGetLastError(), "launching the 8-bit product of few rows");
}

// x8, the scales, and the copy of a weight whose rows are not aligned, in one launch.
template <typename T>
int quantize_of(const void* x, void* values, float* scales, int64_t rows, int64_t width, int64_t stride, const void* w, void* w_out, int64_t outputs, hipStream_t stream) {
  typedef typename T::Storage S;
  const int vec = width % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)values % 8 == 0 && stride % 8 == 0;
  const int64_t copies = w_out == nullptr ? 0 : outputs < 1024 ? outputs : 1024;
  if (!one_launch(rows + copies, 256)) return fail(LIMN_HIP_EUNSUPPORTED, "quantize_rows: %lld rows are out of range, they exceed one launch", (long long)rows);
  hipLaunchKernelGGL((quantize_rows<T>), dim3((unsigned)(rows + copies)), dim3(256), 0, stream, (const S*)x, (signed char*)values, scales, rows, width, stride, vec,
                     (const signed char*)w, (signed char*)w_out, outputs);
  return check_hip(hipGetLastError(), "launching the rounding of rows to 8 bits");
}

int quantize(int dtype, const void* x, void* values, float* scales, int64_t rows, int64_t width, int64_t stride, const void* w, void* w_out, int64_t outputs, hipStream_t stream) {
  return dtype == LIMN_HIP_FLOAT32   ? quantize_of<F32>(x, values, scales, rows, width, stride, w, w_out, outputs, stream)
         : dtype == LIMN_HIP_FLOAT16 ? quantize_of<F16>(x, values, scales, rows, width, stride, w, w_out, outputs, stream)
                                     : quantize_of<BF16>(x, values, scales, rows, width, stride, w, w_out, outputs, stream);
}

// Rows up to which int8_few takes a call: those of one operand. (16 x 4096 x 8192, few and tiles, the rows' rounding with them: 13.4
// and 14.3 us; 16 x 4096 x 2048 11.2 and 13.4; 32 x 4096 x 8192, two operands a wave, 17.3 and 14.9.)
constexpr int64_t FEW = 16;

// The largest tiles where they give every CU a workgroup, the middle ones where they do more than half (1024 x 760 x 2288, 144 of
// them: 16.0 us, 16.9 in the small ones; 512 x 4096 x 4096, 128: 25.5 and 23.2).
int tile_of(const Int8Args& a) { return tiles(a, 256) >= 256 ? 256 : tiles(a, 128) > 128 ? 128 : 64; }

template <typename T>
int product(const Int8Args& a, const signed char* x8, const float* scales, const signed char* w8, int64_t w_stride) {
  if (a.rows <= FEW) return few_of<T, false>(a, x8, scales, w8, w_stride);
  const int m = tile_of(a);
  if (m == 256) return tiles_of<T, 256, 64>(a, x8, scales, w8, w_stride);
  if (m == 128) return tiles_of<T, 128, 128>(a, x8, scales, w8, w_stride);
  return tiles_of<T, 64, 128>(a, x8, scales, w8, w_stride);
}

template <typename T>
int linear(const Int8Args& a) {
  typedef typename T::Storage S;
  const int64_t padded = a.padded();
  signed char* x8 = (signed char*)a.workspace;
  float* scales = (float*)(x8 + align256(a.rows * padded));
  const signed char* w = (const signed char*)a.w;
  const bool copied = needs_copy(w, a.width);
  if (a.rows <= FEW && a.rows * padded <= OWN_BYTES && a.outputs <= OWN_OUTPUTS && !copied && (uintptr_t)a.x % 16 == 0) return few_of<T, true>(a, x8, scales, w, a.width);
  const int64_t blocks = a.rows <= FEW ? (a.outputs + 15) / 16 : tiles(a, tile_of(a));
  if (!one_launch(blocks, 256)) return fail(LIMN_HIP_EUNSUPPORTED, "int8_linear: sizes out of range, %lld workgroups exceed one launch", (long long)blocks);
  if (!copied) {
    const int rc = quantize(a.dtype, a.x, x8, scales, a.rows, a.width, padded, nullptr, nullptr, 0, a.stream);
    return rc != LIMN_HIP_OK ? rc : product<T>(a, x8, scales, w, a.width);
  }
  signed char* const copy = (signed char*)scales + align256(a.rows * 4);
  const int64_t most = copied_outputs(a.width, a.outputs);
  for (int64_t n = 0; n < a.outputs; n += most) {  // the rows' rounding with the first slab's copy
    Int8Args slab = a;
    slab.outputs = std::min(most, a.outputs - n);
    slab.w_scales = a.w_scales + n;
    slab.bias = a.bias == nullptr ? nullptr : (const S*)a.bias + n;
    slab.out = (S*)a.out + n;
    int rc = quantize(a.dtype, a.x, x8, scales, n == 0 ? a.rows : 0, a.width, padded, w + n * a.width, copy, slab.outputs, a.stream);
    if (rc == LIMN_HIP_OK) rc = product<T>(slab, x8, scales, copy, padded);
    if (rc != LIMN_HIP_OK) return rc;
  }
  return LIMN_HIP_OK;
}

int check_sizes(const char* name, int dtype, int64_t rows, int64_t width, int64_t outputs) {
  if (dtype != LIMN_HIP_FLOAT32 && dtype != LIMN_HIP_FLOAT16 && dtype != LIMN_HIP_BFLOAT16)
    return fail(LIMN_HIP_EUNSUPPORTED, "%s: takes float32, float16 or bfloat16, not dtype code %d", name, dtype);
  if (rows < 1 || width < 1 || outputs < 1)
    return fail(LIMN_HIP_EINVAL, "%s: sizes must be positive (rows %lld, width %lld, outputs %lld)", name, (long long)rows, (long long)width, (long long)outputs);
  return LIMN_HIP_OK;
}

constexpr int64_t WIDEST = 1 << 17;  // 2^17 products of at most 127 * 128 stay below 2^31

}  // namespace
}  // namespace limn

using namespace limn;

extern "C" int limn_hip_quantize_rows(const void* x, void* values, void* scales, int dtype, int64_t rows, int64_t width, void* stream) {
  const char* name = "quantize_rows";
  const int rc = check_sizes(name, dtype, rows, width, 1);
  if (rc != LIMN_HIP_OK) return rc;
  if (x == nullptr || values == nullptr || scales == nullptr) return fail(LIMN_HIP_EINVAL, "%s: null buffer", name);
  if ((uintptr_t)x % (dtype == LIMN_HIP_FLOAT32 ? 4 : 2) != 0 || (uintptr_t)scales % 4 != 0)
    return fail(LIMN_HIP_EINVAL, "%s: buffers must be aligned to their element size", name);
  if (!one_launch(rows, 256) || width > ((int64_t)1 << 40) / rows) return fail(LIMN_HIP_EUNSUPPORTED, "%s: sizes out of range", name);
  return quantize(dtype, x, values, (float*)scales, rows, width, width, nullptr, nullptr, 0, (hipStream_t)stream);
}

extern "C" int64_t limn_hip_int8_linear_workspace(int dtype, int64_t rows, int64_t width, int64_t outputs) {
  if (rows < 1 || width < 1 || width > WIDEST || outputs < 1 || rows > 0x7fffffff || outputs > 0x7fffffff) return 0;
  const int64_t padded = (width + PAD - 1) / PAD * PAD;
  return align256(rows * padded) + align256(rows * 4) + copied_outputs(width, outputs) * padded;  // the copy too: a weight's rows may be aligned, its start not
}

extern "C" int limn_hip_int8_linear(const void* x, const void* weight, const void* weight_scales, const void* bias, void* out, int dtype, int64_t rows,
                                    int64_t width, int64_t outputs, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "int8_linear";
  const int rc = check_sizes(name, dtype, rows, width, outputs);
  if (rc != LIMN_HIP_OK) return rc;
  if (x == nullptr || weight == nullptr || weight_scales == nullptr || out == nullptr) return fail(LIMN_HIP_EINVAL, "%s: null buffer", name);
  const uintptr_t size = dtype == LIMN_HIP_FLOAT32 ? 4 : 2;
  if (((uintptr_t)x | (uintptr_t)bias | (uintptr_t)out) % size != 0 || (uintptr_t)weight_scales % 4 != 0)
    return fail(LIMN_HIP_EINVAL, "%s: buffers must be aligned to their element size", name);
  if (width > WIDEST || rows > 0x7fffffff || outputs > 0x7fffffff)
    return fail(LIMN_HIP_EUNSUPPORTED, "%s: sizes out of range (a width of %lld: sums of up to 2^17 products are exact)", name, (long long)width);
  if (workspace_bytes < 0) return fail(LIMN_HIP_EINVAL, "%s: negative workspace size", name);
  if (workspace == nullptr || (uintptr_t)workspace % 16 != 0 || workspace_bytes < limn_hip_int8_linear_workspace(dtype, rows, width, outputs))
    return fail(LIMN_HIP_EINVAL, "%s: needs a workspace of %lld bytes, 16-byte aligned", name, (long long)limn_hip_int8_linear_workspace(dtype, rows, width, outputs));
  const Int8Args a = {x, weight, (const float*)weight_scales, bias, out, dtype, rows, width, outputs, outputs, workspace, (hipStream_t)stream};
  return dtype == LIMN_HIP_FLOAT32 ? linear<F32>(a) : dtype == LIMN_HIP_FLOAT16 ? linear<F16>(a) : linear<BF16>(a);
}
