// Operands of the contraction kernels that go from memory straight into LDS (buffer_load ... lds), in the
// swizzled tiles that matmul.hip describes. Shared by matmul.hip and the cross entropy's products (xent_tiles.hip).
#pragma once

#include "matmul.h"

namespace limn {
namespace {

constexpr int BK = 64;

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

typedef __attribute__((address_space(3))) void lds_void;

// the s_waitcnt immediate that waits for every outstanding vector memory operation (vmcnt 0) and
// leaves the other counters free
constexpr int WAIT_VMEM = 0x0F70;

// One operand's DMA copy into a swizzled LDS tile, and its MFMA operand reads.
template <int ROWS, bool KCONTIG, int WAVES>
struct DmaOperand {
  static constexpr int RB = KCONTIG ? BK * 2 : ROWS * 2;  // bytes per LDS row
  static constexpr int BYTES = (KCONTIG ? ROWS : BK) * RB;
  static constexpr int PASSES = BYTES / (1024 * WAVES);   // 1 KB DMA instructions per wave per stage
  static constexpr int RPI = 1024 / RB;                   // LDS rows one DMA instruction fills
  static constexpr int READS = KCONTIG ? 1 : 2;           // LDS reads per MFMA operand
  static_assert(PASSES * 1024 * WAVES == BYTES, "a stage is a whole number of DMA passes");
  static __device__ __forceinline__ int swizzle(int r) { return KCONTIG ? (r >> 1) & 7 : (r & 3) << 2; }

  const char* base;
  int64_t extent, step, first;  // bytes from base the operand spans; bytes per stage; first stage
  int voff[PASSES];

  __device__ __forceinline__ DmaOperand(const u16* b, int64_t rows, int64_t depth, int64_t stride, int64_t row0,
                                        int64_t k_lo, int wave, int lane) {
    base = (const char*)b;
    extent = 2 * (KCONTIG ? (rows - 1) * stride + depth : (depth - 1) * stride + rows);
    step = KCONTIG ? 2 * BK : 2 * BK * stride;
    first = k_lo / BK;
#pragma unroll
    for (int q = 0; q < PASSES; q++) {
      // lane `lane` of this wave's q-th instruction fills position `pos` of LDS row r
      const int r = (q * WAVES + wave) * RPI + lane / (RB / 16), pos = lane % (RB / 16);
      const int c = pos ^ swizzle(r);
      voff[q] = KCONTIG ? (int)(((row0 + r) * stride + c * 8) * 2) : (int)((r * stride + row0 + c * 8) * 2);
    }
  }

  // this wave's share of stage st into `tile`; a stage past the end reads zeros (or the next
  // slice's k) into the idle buffer, where nothing reads it
  __device__ __forceinline__ void copy(char* tile, int st, int wave) const {
    const int64_t off = (first + st) * step, left = extent - off;
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)(base + off), (short)0, (int)(left > 0 ? left : 0), 0x00020000);
#pragma unroll
    for (int q = 0; q < PASSES; q++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(tile + (q * WAVES + wave) * 1024), 16, voff[q], 0, 0, 0);
  }

  // per-lane read offsets for the T 32-row blocks a wave multiplies, starting at row `row0`: by
  // k step for a k-contiguous tile (the swizzle varies with k), by block otherwise
  template <int T>
  __device__ __forceinline__ void offsets(int row0, int lane, int* rd) const {
    if (KCONTIG) {
      const int r = lane & 31, h = lane >> 5;
#pragma unroll
      for (int kk = 0; kk < BK / 16; kk++) rd[kk] = (row0 + r) * RB + (((2 * kk + h) ^ swizzle(r)) & 7) * 16;
    } else {
      const int g = lane >> 4, i = lane & 15, k = 8 * (g >> 1) + (i >> 2);
#pragma unroll
      for (int t = 0; t < T; t++) {
        const int col = row0 + t * 32 + 16 * (g & 1) + 4 * (i & 3);
        rd[t] = k * RB + ((col >> 3) ^ swizzle(k)) * 16 + (col & 7) * 2;
      }
    }
  }

  // the MFMA operand of block t at k step kk: lane l gets X[row0 + 32 t + l % 32][16 kk + 8 (l / 32) + j]
  __device__ __forceinline__ u16x8 operand(const char* tile, const int* rd, int t, int kk) const {
    if (KCONTIG) return *(const u16x8*)(tile + rd[kk] + t * 32 * RB);
    // a transposing read gives lane i of each 16-lane group item j from the 8 bytes lane 4j + i/4
    // addresses, element i % 4: lane r addresses k row 16 kk + 8 (l / 32) + r / 4 (+ 4 for the
    // second read), columns row0 + 32 t + 16 ((l / 16) % 2) + 4 (r % 4)
    const char* p = tile + rd[t] + kk * 16 * RB;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)p);
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p + 4 * RB));
    return __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

template <int BM>
struct DmaTile {
  static constexpr int WAVES = BM == 256 ? 8 : 4;
  static constexpr int WN = WAVES / 2;  // waves along n; 2 along m
};

}  // namespace
}  // namespace limn
