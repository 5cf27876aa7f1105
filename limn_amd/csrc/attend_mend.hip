// Beside the tiled kernels of attention with score rules (attend_mfma.h, attend_parts.h): the ranges of documents that
// let them skip tiles, and the blocks that hidden infinities or NaN spoiled, computed again in float.

#include "attend_fast.h"
#include "attend_general.h"

namespace limn {
namespace {

// The least and greatest document of each 32 positions, padding and positions past the live keys left out
// (0x7fffffff and 0, an empty range, if there is nothing else), and the document of all 32, or -2.
__global__ __launch_bounds__(256) void attend_ranges(RuleArgs ra, int4* __restrict__ ranges, int64_t batch, int granules) {
  const int64_t id = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5), b = id / granules;
  if (b >= batch) return;  // a half wave at a time: the shuffles below stay inside it
  const int g = (int)(id - b * granules), n = threadIdx.x & 31, p = g * 32 + n;
  const int len = ra.lengths ? ra.lengths[b] : ra.t_k;
  int doc = -1;
  if (p < ra.t_k && p < len) doc = ra.documents[b * ra.t_k + p];
  int lo = doc < 0 ? 0x7fffffff : doc, hi = doc < 0 ? 0 : doc, none = doc < 0;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    lo = min(lo, __shfl_xor(lo, m));
    hi = max(hi, __shfl_xor(hi, m));
    none |= __shfl_xor(none, m);
  }
  if (n == 0) ranges[id] = make_int4(lo, hi, lo == hi && !none ? lo : -2, 0);
}

// delta = rowsum(dout * out), 16 lanes a row
template <typename T>
__global__ __launch_bounds__(256) void attend_delta(FastArgs g, int64_t rows) {
  const int64_t row = blockIdx.x * (int64_t)16 + (threadIdx.x >> 4);
  if (row >= rows) return;  // 16 lanes at a time: the shuffles below stay inside them
  const int d = (threadIdx.x & 15) * 8;
  float x = 0.f;
  if (d < g.hd) {
    const u16x8 a = *(const u16x8*)(g.dout + row * g.hd + d), b = *(const u16x8*)(g.out + row * g.hd + d);
#pragma unroll
    for (int e = 0; e < 8; e++) x = fmaf(T::unpack(a[e]), T::unpack(b[e]), x);
  }
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) x += __shfl_xor(x, m);
  if (d == 0) g.delta[row] = x;
}

// The flagged blocks among those of this workgroup (every gridDim.x-th), found 256 flags at a time.
template <typename F>
__device__ __forceinline__ void each_odd(const int* odd, int64_t blocks, F f) {
  for (int64_t first = blockIdx.x; first < blocks; first += (int64_t)gridDim.x * 256) {
    const int64_t mine = first + (int64_t)threadIdx.x * gridDim.x;
    if (!__syncthreads_or(mine < blocks && odd[mine] != 0)) continue;
    for (int j = 0; j < 256; j++) {
      const int64_t id = first + (int64_t)j * gridDim.x;
      if (id >= blocks) break;
      if (odd[id] != 0) f(id);  // the same for every thread
    }
  }
}

template <typename T, int DT>
__global__ __launch_bounds__(GEN_THREADS, 1) void attend_mend_fwd(FastArgs g, RuleArgs ra, int64_t blocks) {
  __shared__ float lds[GEN_LDS];
  const int64_t nqb = (ra.t_q + ATT_ROWS - 1) / ATT_ROWS;
  each_odd(g.odd, blocks, [&](int64_t id) {
    const int64_t bh = id / nqb, b = bh / g.heads;
    const int head = (int)(bh - b * g.heads), q0 = (int)(id - bh * nqb) * ATT_ROWS;
    const GenFwd gen = {g.q, g.k, g.v, g.o0, g.lse, nullptr, nullptr, g.batch, g.heads, g.kv_heads, g.hd, g.hd, 1, 1};
    for (int j = 0; j < ATT_ROWS && q0 + j < ra.t_q; j += 32)
      gen_fwd_block<T, DT>(gen, ra, RowMap{1, head, ra.t_q}, b, head / (g.heads / g.kv_heads), q0 + j, 0, lds);
  });
}

// Both of the backward's passes: two kernels were 2 us more where there is nothing to mend.
template <typename T, int DT>
__global__ __launch_bounds__(GEN_THREADS, 1) void attend_mend_bwd(FastArgs g, FastArgs kv, RuleArgs ra, int64_t blocks, int64_t kv_blocks) {
  __shared__ float lds[GEN_LDS];
  const int64_t nqb = (ra.t_q + ATT_ROWS - 1) / ATT_ROWS, nkb = (ra.t_k + ATT_ROWS - 1) / ATT_ROWS;
  const int group = g.heads / g.kv_heads;
  const GenBwd gen = {g.q, g.k, g.v, g.out, g.dout, g.lse_in, g.delta, g.o0, kv.o0, kv.o1, g.heads, g.kv_heads, g.hd, g.hd, 1, g.scale};
  each_odd(g.odd, blocks, [&](int64_t id) {
    const int64_t bh = id / nqb, b = bh / g.heads;
    const int head = (int)(bh - b * g.heads), q0 = (int)(id - bh * nqb) * ATT_ROWS;
    for (int j = 0; j < ATT_ROWS && q0 + j < ra.t_q; j += 32) gen_dq_block<T, DT>(gen, ra, RowMap{1, head, ra.t_q}, b, head / group, q0 + j, false, lds);
  });
  each_odd(kv.odd, kv_blocks, [&](int64_t id) {
    const int64_t bk = id / nkb, b = bk / g.kv_heads;
    const int kvh = (int)(bk - b * g.kv_heads), k0 = (int)(id - bk * nkb) * ATT_ROWS;
    for (int j = 0; j < ATT_ROWS && k0 + j < ra.t_k; j += 32) gen_dkv_block<T, DT, (DT <= 2)>(gen, ra, RowMap{group, kvh * group, group * ra.t_q}, b, kvh, k0 + j, lds);
  });
}

// The forward's tiles of 32 packed rows, each computed again if one of its results is not finite.
template <typename T, int DT>
__global__ __launch_bounds__(GEN_THREADS, 1) void attend_mend_rows(GenFwd g, RuleArgs ra, int64_t tiles, int row_tiles) {
  __shared__ float lds[GEN_LDS];
  const int group = g.heads / g.kv_heads, rows = group * ra.t_q;
  for (int64_t id = blockIdx.x; id < tiles; id += gridDim.x) {
    const int64_t bk = id / row_tiles, b = bk / g.kv_heads;
    const int kvh = (int)(bk - b * g.kv_heads), row0 = (int)(id - bk * row_tiles) * 32;
    const RowMap map = {group, kvh * group, rows};
    bool odd = false;
    for (int i = threadIdx.x; i < 32 * g.hd_v; i += GEN_THREADS) {
      const int row = row0 + i / g.hd_v;
      if (row < rows) odd |= !gen_finite(T::load((const u16*)g.out + b * g.heads * (int64_t)ra.t_q * g.hd_v + map.at(row, ra.t_q, g.hd_v), i % g.hd_v));
    }
    if (__syncthreads_or(odd)) gen_fwd_block<T, DT>(g, ra, map, b, kvh, row0, 0, lds);
  }
}

constexpr int64_t MEND_GROUPS = 256;

unsigned mend_grid(int64_t blocks) { return (unsigned)(blocks < MEND_GROUPS ? blocks : MEND_GROUPS); }

template <typename T, int DT>
int mend_fwd(const FastArgs& g, const RuleArgs& ra, hipStream_t stream) {
  const int64_t blocks = g.batch * g.heads * ((ra.t_q + ATT_ROWS - 1) / ATT_ROWS);
  hipLaunchKernelGGL((attend_mend_fwd<T, DT>), dim3(mend_grid(blocks)), dim3(GEN_THREADS), 0, stream, g, ra, blocks);
  return check_hip(hipGetLastError(), "launching attention's mending");
}

template <typename T, int DT>
int mend_bwd(const FastArgs& g, const FastArgs& kv, const RuleArgs& ra, hipStream_t stream) {
  const int64_t blocks = g.batch * g.heads * ((ra.t_q + ATT_ROWS - 1) / ATT_ROWS), kv_blocks = g.batch * g.kv_heads * ((ra.t_k + ATT_ROWS - 1) / ATT_ROWS);
  hipLaunchKernelGGL((attend_mend_bwd<T, DT>), dim3(mend_grid(blocks > kv_blocks ? blocks : kv_blocks)), dim3(GEN_THREADS), 0, stream, g, kv, ra, blocks, kv_blocks);
  return check_hip(hipGetLastError(), "launching attention's mending");
}

template <typename T, int DT>
int mend_rows(const AttendArgs& a) {
  const int64_t row_tiles = (a.group() * a.t_q + 31) / 32, tiles = a.batch * a.kv_heads * row_tiles;
  const GenFwd g = {a.q, a.k, a.v, a.o0, (float*)a.o1, nullptr, nullptr, a.batch, (int)a.heads, (int)a.kv_heads, (int)a.hd, (int)a.hd_v, 1, 1};
  hipLaunchKernelGGL((attend_mend_rows<T, DT>), dim3((unsigned)(tiles < 1024 ? tiles : 1024)), dim3(GEN_THREADS), 0, a.stream, g, rule_args(a), tiles, (int)row_tiles);
  return check_hip(hipGetLastError(), "launching attention's mending");
}

}  // namespace

int launch_attend_mend_rows(const AttendArgs& a) {
  if (a.dtype == LIMN_HIP_BFLOAT16) return a.hd <= 64 ? mend_rows<BF16, 2>(a) : mend_rows<BF16, 4>(a);
  return a.hd <= 64 ? mend_rows<F16, 2>(a) : mend_rows<F16, 4>(a);
}

int launch_attend_ranges(const RuleArgs& ra, int4* ranges, int64_t batch, int granules, hipStream_t stream) {
  const int64_t blocks = (batch * granules + 7) / 8;
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "attend: %lld workgroups exceed one launch", (long long)blocks);
  hipLaunchKernelGGL(attend_ranges, dim3((unsigned)blocks), dim3(256), 0, stream, ra, ranges, batch, granules);
  return check_hip(hipGetLastError(), "launching the documents' ranges");
}

int launch_attend_delta(const FastArgs& g, int64_t rows, int dtype, hipStream_t stream) {
  const int64_t blocks = (rows + 15) / 16;
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "attend: %lld workgroups exceed one launch", (long long)blocks);
  if (dtype == LIMN_HIP_BFLOAT16)
    hipLaunchKernelGGL((attend_delta<BF16>), dim3((unsigned)blocks), dim3(256), 0, stream, g, rows);
  else
    hipLaunchKernelGGL((attend_delta<F16>), dim3((unsigned)blocks), dim3(256), 0, stream, g, rows);
  return check_hip(hipGetLastError(), "launching attention's row sums");
}

int launch_attend_mend_fwd(const FastArgs& g, const RuleArgs& ra, int dtype, hipStream_t stream) {
  if (dtype == LIMN_HIP_FLOAT32) return g.hd <= 64 ? mend_fwd<F32, 2>(g, ra, stream) : mend_fwd<F32, 4>(g, ra, stream);
  if (dtype == LIMN_HIP_BFLOAT16) return g.hd <= 64 ? mend_fwd<BF16, 2>(g, ra, stream) : mend_fwd<BF16, 4>(g, ra, stream);
  return g.hd <= 64 ? mend_fwd<F16, 2>(g, ra, stream) : mend_fwd<F16, 4>(g, ra, stream);
}

int launch_attend_mend_bwd(const FastArgs& g, const FastArgs& kv, const RuleArgs& ra, int dtype, hipStream_t stream) {
  if (dtype == LIMN_HIP_FLOAT32) return g.hd <= 64 ? mend_bwd<F32, 2>(g, kv, ra, stream) : mend_bwd<F32, 4>(g, kv, ra, stream);
  if (dtype == LIMN_HIP_BFLOAT16) return g.hd <= 64 ? mend_bwd<BF16, 2>(g, kv, ra, stream) : mend_bwd<BF16, 4>(g, kv, ra, stream);
  return g.hd <= 64 ? mend_bwd<F16, 2>(g, kv, ra, stream) : mend_bwd<F16, 4>(g, kv, ra, stream);
}

}  // namespace limn
