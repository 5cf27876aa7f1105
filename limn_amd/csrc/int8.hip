// A linear layer in 8-bit integers (include/limn_hip.h, limn_hip_int8_linear) and the bringing of rows to 8 bits
// (limn_hip_quantize_rows):
//
//   s = max(max |x| / 127, 2^-126),  x8 = round(x / s) (ties to even),  y = (x8 . w8) s scale + bias.
//
// Sums of products are whole numbers in 32 bits, exact up to 2^17 terms of 127 * 128. The product runs on
// v_mfma_i32_32x32x32_i8 in the tiles of matmul.hip's DMA kernel, with bytes where that has 16-bit elements: rows of 128
// bytes a stage, 16-byte chunk c of LDS row r at position c ^ ((r >> 1) & 7), copied straight to LDS, the next stage in
// flight while one is multiplied. Rows of x8 are padded with zeros to whole stages, so what a stage holds of a weight's next
// row is multiplied by 0; rows past an operand's end read as zeros.

#include "common.h"

#include <math.h>

namespace limn {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int STAGE = 128;          // bytes of a row that a stage holds
constexpr int WAIT_VMEM = 0x0F70;   // s_waitcnt: every vector memory operation done, the other counters free

struct Int8Args {
  const void* x;
  const void* w;
  const float* w_scales;
  const void* bias;  // of x's type, or nullptr
  void* out;
  int dtype;
  int64_t rows, width, outputs;
  void* workspace;
  hipStream_t stream;
  int64_t padded() const { return (width + STAGE - 1) / STAGE * STAGE; }
};

constexpr int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The copy of the weight with aligned rows that a call needs where its rows are not.
bool needs_copy(const void* w, int64_t width) { return width % 16 != 0 || (uintptr_t)w % 16 != 0; }

// A workgroup a row: its largest magnitude, then its numbers, `stride` bytes a row, zeros behind the width. A row with an
// infinity or a NaN gets the scale NaN and zeros.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows(const typename T::Storage* __restrict__ x, signed char* __restrict__ out, float* __restrict__ scales,
                                                     int64_t width, int64_t stride) {
  __shared__ float tops[4];
  const typename T::Storage* row = x + blockIdx.x * width;
  float top = 0.f, odd = 0.f;
  for (int64_t i = threadIdx.x; i < width; i += 256) {
    const float v = T::load(row, i);
    top = fmaxf(top, fabsf(v));
    odd = fmaf(v, 0.f, odd);  // NaN once an infinity or a NaN was there
  }
  if (odd != odd) top = __builtin_inff();
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const bool fine = top < __builtin_inff();
  const float s = fmaxf(top / 127.f, 0x1p-126f);
  if (threadIdx.x == 0) scales[blockIdx.x] = fine ? s : __builtin_nanf("");
  signed char* o = out + blockIdx.x * stride;
  for (int64_t i = threadIdx.x; i < stride; i += 256) o[i] = fine && i < width ? (signed char)(int)rintf(T::load(row, i) / s) : 0;
}

__global__ __launch_bounds__(256) void pad_rows(const signed char* __restrict__ w, signed char* __restrict__ out, int64_t width, int64_t stride) {
  for (int64_t i = threadIdx.x; i < stride; i += 256) out[blockIdx.x * stride + i] = i < width ? w[blockIdx.x * width + i] : 0;
}

// One operand's tile of ROWS rows from row0 on: the copy of a stage to LDS, and the matrix instruction's operands.
template <int ROWS, int WAVES>
struct Tile {
  static constexpr int BYTES = ROWS * STAGE, PASSES = BYTES / (1024 * WAVES);
  static __device__ __forceinline__ int swizzle(int r) { return (r >> 1) & 7; }
  const char* base;
  int64_t extent;  // bytes from base to the operand's end
  int voff[PASSES];
  __device__ __forceinline__ Tile(const signed char* p, int64_t rows, int64_t stride, int64_t row0, int wave, int lane) {
    base = (const char*)p + row0 * stride;
    extent = (rows - row0) * stride;
#pragma unroll
    for (int q = 0; q < PASSES; q++) {
      const int r = (q * WAVES + wave) * 8 + lane / 8;
      voff[q] = (int)(r * stride) + ((lane % 8) ^ swizzle(r)) * 16;
    }
  }
  __device__ __forceinline__ void copy(char* tile, int stage, int wave) const {
    const int64_t off = (int64_t)stage * STAGE, left = extent - off;
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)(base + off), (short)0, (int)(left < 0 ? 0 : left < 0x7fffffff ? left : 0x7fffffff), 0x00020000);
#pragma unroll
    for (int q = 0; q < PASSES; q++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(tile + (q * WAVES + wave) * 1024), 16, voff[q], 0, 0, 0);
  }
  // lane l: bytes 32 kk + 16 (l / 32) .. + 15 of row row0 + l % 32; kk a place in rd
  static __device__ __forceinline__ void offsets(int row0, int lane, int* rd) {
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int kk = 0; kk < 4; kk++) rd[kk] = (row0 + r) * STAGE + (((2 * kk + h) ^ swizzle(r)) & 7) * 16;
  }
  static __device__ __forceinline__ i32x4 operand(const char* tile, const int* rd, int t, int kk) { return *(const i32x4*)(tile + rd[kk] + t * 32 * STAGE); }
};

// out[m, n] = (x8[m] . w8[n]) s[m] scale[n] + bias[n], one rounding a step in float, rounded to the type at the end.
template <typename T, int BM>
__global__ __launch_bounds__(BM == 256 ? 512 : 256, 2) void int8_tiles(const signed char* __restrict__ x8, const float* __restrict__ scales, const signed char* __restrict__ w8,
                                                                       int64_t w_stride, Int8Args a) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr int WAVES = BM == 256 ? 8 : 4, WN = WAVES / 2, WTM = BM / 2, WTN = BM / WN, TM = WTM / 32, TN = WTN / 32;
  typedef Tile<BM, WAVES> O;
  __shared__ __attribute__((aligned(1024))) char A0[O::BYTES];
  __shared__ __attribute__((aligned(1024))) char A1[O::BYTES];
  __shared__ __attribute__((aligned(1024))) char B0[O::BYTES];
  __shared__ __attribute__((aligned(1024))) char B1[O::BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n32 = lane & 31;
  const int wm = wave / WN, wn = wave % WN;
  const int64_t tiles_n = (a.outputs + BM - 1) / BM, tiles_m = (a.rows + BM - 1) / BM;
  int64_t id = blockIdx.x;
  if (gridDim.x % 8 == 0) id = (id % 8) * (gridDim.x / 8) + id / 8;  // an XCD's workgroups: a run of tiles, 4 tile rows at a time
  constexpr int64_t GROUP = 4;
  const int64_t group = id / (GROUP * tiles_n), first = group * GROUP, live = tiles_m - first < GROUP ? tiles_m - first : GROUP;
  const int64_t m0 = (first + (id - group * GROUP * tiles_n) % live) * BM, n0 = (id - group * GROUP * tiles_n) / live * BM;
  const int64_t padded = (a.width + STAGE - 1) / STAGE * STAGE;
  const int stages = (int)(padded / STAGE);

  i32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
  const O da(x8, a.rows, padded, m0, wave, lane), db(w8, a.outputs, w_stride, n0, wave, lane);
  int rda[4], rdb[4];
  O::offsets(wm * WTM, lane, rda);
  O::offsets(wn * WTN, lane, rdb);
  auto stage = [&](const char* at, const char* bt, char* an, char* bn, int st) __attribute__((always_inline)) {
    da.copy(an, st + 1, wave);
    db.copy(bn, st + 1, wave);
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
      i32x4 av[TM], bv[TN];
#pragma unroll
      for (int i = 0; i < TM; i++) av[i] = O::operand(at, rda, i, kk);
#pragma unroll
      for (int j = 0; j < TN; j++) bv[j] = O::operand(bt, rdb, j, kk);
      // the weight's operand first: a lane then holds 4 consecutive outputs of a row
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bv[j], av[i], acc[i][j], 0, 0, 0);
    }
    __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
    __syncthreads();
  };
  da.copy(A0, 0, wave);
  db.copy(B0, 0, wave);
  __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
  __syncthreads();
  for (int st = 0; st < stages; st += 2) {
    stage(A0, B0, A1, B1, st);
    if (st + 1 < stages) stage(A1, B1, A0, B0, st + 1);
  }
  typename T::Storage* out = (typename T::Storage*)a.out;
  const typename T::Storage* bias = (const typename T::Storage*)a.bias;
#pragma unroll
  for (int i = 0; i < TM; i++) {
    const int64_t row = m0 + wm * WTM + i * 32 + n32;
    const float s = row < a.rows ? scales[row] : 0.f;
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int64_t col = n0 + wn * WTN + j * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
        if (row >= a.rows || col >= a.outputs) continue;
        float y = (float)acc[i][j][e] * a.w_scales[col] * s;  // the scale of x last: it may be as large as x
        if (bias != nullptr) y += T::load(bias, col);
        T::store(out, row * a.outputs + col, y);
      }
  }
#endif
}

template <typename T, int BM>
int tiles_of(const Int8Args& a, const signed char* x8, const float* scales, const signed char* w8, int64_t w_stride) {
  const int64_t blocks = ((a.rows + BM - 1) / BM) * ((a.outputs + BM - 1) / BM);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "int8_linear: %lld workgroups exceed one launch", (long long)blocks);
  hipLaunchKernelGGL((int8_tiles<T, BM>), dim3((unsigned)blocks), dim3(BM == 256 ? 512 : 256), 0, a.stream, x8, scales, w8, w_stride, a);
  return check_hip(hipGetLastError(), "launching the 8-bit product");
}

template <typename T>
int quantize_of(const void* x, void* values, float* scales, int64_t rows, int64_t width, int64_t stride, hipStream_t stream) {
  hipLaunchKernelGGL((quantize_rows<T>), dim3((unsigned)rows), dim3(256), 0, stream, (const typename T::Storage*)x, (signed char*)values, scales, width, stride);
  return check_hip(hipGetLastError(), "launching the rounding of rows to 8 bits");
}

int quantize(int dtype, const void* x, void* values, float* scales, int64_t rows, int64_t width, int64_t stride, hipStream_t stream) {
  return dtype == LIMN_HIP_FLOAT32   ? quantize_of<F32>(x, values, scales, rows, width, stride, stream)
         : dtype == LIMN_HIP_FLOAT16 ? quantize_of<F16>(x, values, scales, rows, width, stride, stream)
                                     : quantize_of<BF16>(x, values, scales, rows, width, stride, stream);
}

template <typename T>
int linear(const Int8Args& a) {
  const int64_t padded = a.padded();
  signed char* x8 = (signed char*)a.workspace;
  float* scales = (float*)(x8 + align256(a.rows * padded));
  const signed char* w8 = (const signed char*)a.w;
  int64_t w_stride = a.width;
  int rc = quantize(a.dtype, a.x, x8, scales, a.rows, a.width, padded, a.stream);
  if (rc != LIMN_HIP_OK) return rc;
  if (needs_copy(a.w, a.width)) {
    signed char* copy = (signed char*)scales + align256(a.rows * 4);
    hipLaunchKernelGGL(pad_rows, dim3((unsigned)a.outputs), dim3(256), 0, a.stream, w8, copy, a.width, padded);
    rc = check_hip(hipGetLastError(), "launching the copy of an 8-bit weight");
    if (rc != LIMN_HIP_OK) return rc;
    w8 = copy;
    w_stride = padded;
  }
  const int64_t t256 = ((a.rows + 255) / 256) * ((a.outputs + 255) / 256);
  return t256 >= 256 ? tiles_of<T, 256>(a, x8, scales, w8, w_stride) : tiles_of<T, 128>(a, x8, scales, w8, w_stride);
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
  if (rows > 0x7fffffff || width > ((int64_t)1 << 40) / rows) return fail(LIMN_HIP_EUNSUPPORTED, "%s: sizes out of range", name);
  return quantize(dtype, x, values, (float*)scales, rows, width, width, (hipStream_t)stream);
}

extern "C" int64_t limn_hip_int8_linear_workspace(int dtype, int64_t rows, int64_t width, int64_t outputs) {
  if (rows < 1 || width < 1 || width > WIDEST || outputs < 1 || rows > 0x7fffffff || outputs > 0x7fffffff) return 0;
  const int64_t padded = (width + STAGE - 1) / STAGE * STAGE;
  return align256(rows * padded) + align256(rows * 4) + outputs * padded;  // the copy too: a weight's rows may be aligned, its start not
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
  const Int8Args a = {x, weight, (const float*)weight_scales, bias, out, dtype, rows, width, outputs, workspace, (hipStream_t)stream};
  return dtype == LIMN_HIP_FLOAT32 ? linear<F32>(a) : dtype == LIMN_HIP_FLOAT16 ? linear<F16>(a) : linear<BF16>(a);
}
