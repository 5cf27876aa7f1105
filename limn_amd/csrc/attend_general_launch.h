// Kernels and launches of attend_general.h for one storage type; each attend_general_*.hip instantiates it
// for one (they compile in parallel).
#pragma once

#include "attend_general.h"

namespace limn {
namespace {

template <typename T, int DT>
__global__ __launch_bounds__(GEN_THREADS, 1) void attend_general_fwd(GenFwd g, RuleArgs ra) {
  __shared__ float lds[GEN_LDS];
  const RowMap map = {g.heads / g.kv_heads, 0, g.heads / g.kv_heads * ra.t_q};
  const int row_tiles = (map.rows + 31) / 32;
  const int split = (int)(blockIdx.x % g.splits);
  int64_t id = blockIdx.x / g.splits;
  const int rt = row_tiles - 1 - (int)(id % row_tiles);  // causal: the longest rows first
  id /= row_tiles;
  const int kvh = (int)(id % g.kv_heads);
  RowMap here = map;
  here.head0 = kvh * map.group;
  gen_fwd_block<T, DT>(g, ra, here, id / g.kv_heads, kvh, rt * 32, split, lds);
}

template <typename T, int DT>
__global__ __launch_bounds__(GEN_THREADS, 1) void attend_general_dq(GenBwd g, RuleArgs ra) {
  __shared__ float lds[GEN_LDS];
  const int group = g.heads / g.kv_heads, rows = group * ra.t_q, row_tiles = (rows + 31) / 32;
  int64_t id = blockIdx.x;
  const int rt = row_tiles - 1 - (int)(id % row_tiles);
  id /= row_tiles;
  const int kvh = (int)(id % g.kv_heads);
  gen_dq_block<T, DT>(g, ra, RowMap{group, kvh * group, rows}, id / g.kv_heads, kvh, rt * 32, true, lds);
}

template <typename T, int DT>
__global__ __launch_bounds__(GEN_THREADS, 1) void attend_general_dkv(GenBwd g, RuleArgs ra) {
  __shared__ float lds[GEN_LDS];
  const int group = g.heads / g.kv_heads, key_tiles = (ra.t_k + 31) / 32;
  int64_t id = blockIdx.x;
  const int kt = (int)(id % key_tiles);  // causal: the first keys are seen by the most rows
  id /= key_tiles;
  const int kvh = (int)(id % g.kv_heads);
  gen_dkv_block<T, DT>(g, ra, RowMap{group, kvh * group, group * ra.t_q}, id / g.kv_heads, kvh, kt * 32, lds);
}

// whether rows of `width` elements from `p` allow loads of 4 elements
template <typename T>
bool gen_vec(const void* p, int64_t width) {
  return width % 4 == 0 && (uintptr_t)p % (4 * sizeof(typename T::Storage)) == 0;
}

template <typename T, int DT>
int launch_gen_fwd(const AttendArgs& a, int64_t splits) {
  const int64_t rows = a.group() * a.t_q, blocks = splits * a.batch * a.kv_heads * ((rows + 31) / 32);
  if (blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "attend: %lld workgroups exceed one launch", (long long)blocks);
  float* totals = nullptr;
  float* stats = nullptr;
  if (splits > 1) {
    totals = (float*)a.workspace;
    stats = (float*)((char*)a.workspace + attend_align(splits * a.batch * a.kv_heads * rows * a.hd_v * 4));
  }
  const int vec = gen_vec<T>(a.q, a.hd) && gen_vec<T>(a.k, a.hd);
  GenFwd g = {a.q, a.k, a.v, a.o0, (float*)a.o1, totals, stats, a.batch, (int)a.heads, (int)a.kv_heads, (int)a.hd, (int)a.hd_v, vec, (int)splits};
  hipLaunchKernelGGL((attend_general_fwd<T, DT>), dim3((unsigned)blocks), dim3(GEN_THREADS), 0, a.stream, g, rule_args(a));
  const int rc = check_hip(hipGetLastError(), "launching attention");
  return rc != LIMN_HIP_OK || splits == 1 ? rc : launch_attend_join(a, totals, stats, splits, 0.f);
}

template <typename T, int DT>
int launch_gen_bwd(const AttendArgs& a) {
  const int64_t rows = a.group() * a.t_q, heads = a.batch * a.kv_heads;
  const int64_t row_blocks = heads * ((rows + 31) / 32), key_blocks = heads * ((a.t_k + 31) / 32);
  if (row_blocks > 0x7fffffff || key_blocks > 0x7fffffff) return fail(LIMN_HIP_EUNSUPPORTED, "attend: too many workgroups for one launch");
  const bool vec = gen_vec<T>(a.q, a.hd) && gen_vec<T>(a.k, a.hd) && gen_vec<T>(a.v, a.hd_v) && gen_vec<T>(a.out, a.hd_v) && gen_vec<T>(a.dout, a.hd_v);
  GenBwd g = {a.q, a.k, a.v, a.out, a.dout, a.lse, (float*)a.workspace, a.o0, a.o1, a.o2, (int)a.heads, (int)a.kv_heads, (int)a.hd, (int)a.hd_v, vec, (float)a.scale};
  hipLaunchKernelGGL((attend_general_dq<T, DT>), dim3((unsigned)row_blocks), dim3(GEN_THREADS), 0, a.stream, g, rule_args(a));
  int rc = check_hip(hipGetLastError(), "launching attention's dQ pass");
  if (rc != LIMN_HIP_OK) return rc;
  hipLaunchKernelGGL((attend_general_dkv<T, DT>), dim3((unsigned)key_blocks), dim3(GEN_THREADS), 0, a.stream, g, rule_args(a));
  return check_hip(hipGetLastError(), "launching attention's dK/dV pass");
}

template <typename T>
int gen_fwd(const AttendArgs& a, int64_t splits) {
  const int64_t d = a.hd > a.hd_v ? a.hd : a.hd_v;
  if (d <= 32) return launch_gen_fwd<T, 1>(a, splits);
  if (d <= 64) return launch_gen_fwd<T, 2>(a, splits);
  if (d <= 128) return launch_gen_fwd<T, 4>(a, splits);
  return launch_gen_fwd<T, 8>(a, splits);
}

template <typename T>
int gen_bwd(const AttendArgs& a) {
  const int64_t d = a.hd > a.hd_v ? a.hd : a.hd_v;
  if (d <= 32) return launch_gen_bwd<T, 1>(a);
  if (d <= 64) return launch_gen_bwd<T, 2>(a);
  if (d <= 128) return launch_gen_bwd<T, 4>(a);
  return launch_gen_bwd<T, 8>(a);
}

}  // namespace
}  // namespace limn
