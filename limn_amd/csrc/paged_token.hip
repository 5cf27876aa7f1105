// Attention over a paged cache for sequences of few new tokens: one that was drawn last, a few that are tried at once. Half
// widths of hd a multiple of 8 up to 128, float32 of a multiple of 4, 16-byte aligned rows.
//
// What bounds it is reading the live keys and values once, and everything is laid out for that:
//  - the queries of every head that shares a key head are rows of one tile (16 NR packed rows i * group + head), so keys
//    and values are read once for all of them;
//  - a wave takes 32 keys at a time and reads them from memory straight into matrix operands, no LDS and no barrier in the
//    loop. K: lane (n = lane % 16, g = lane / 16) reads 16 bytes of keys n and 16 + n at a time; V: W = D / 16 dims from W n
//    on (value_dim) of keys 4 g + j and 16 + 4 g + j. S^T = K Q^T leaves exactly those keys' weights in the lane, so they are the second
//    product's operand as they stand. Half widths multiply by v_mfma_f32_16x16x32, float32 by v_mfma_f32_16x16x4_f32;
//  - a lane looks up the place of one key of 32 in the table, a tile ahead, and gets the places of the keys it reads from
//    the other lanes: pages of any size cost the same;
//  - the new tokens' keys and values are read where the caller has them, and put in their places by the workgroups of the
//    first part, so one launch does both. Only among them a query may not see a key;
//  - long caches are cut into parts over workgroups, joined by a second kernel in the order of the parts.
//
// Hidden keys' values must not reach a row: a weight of 0 times an infinity or a NaN is NaN. Tiles
// with keys that some rows do not see are looked over (see give_back).

#include "paged_fast.h"
#include "paged_reads.h"

namespace limn {
namespace {

constexpr int KEYS = 32;  // keys a wave takes at a time

// the 4 lanes of a column (lanes n, n + 16, n + 32, n + 48) combined
__device__ __forceinline__ float col_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float col_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// How a type's bytes become operands: K in chunks of 16 bytes, V in chunks of W elements a key.
template <typename T, int W>
struct Operands {
  typedef u16 S;
  static constexpr int PER = 8;  // elements of 16 bytes
  struct Chunk {
    u16x8 x;
  };
  struct Values {
    u16 x[W];
  };
  static __device__ __forceinline__ f32x4 mfma(u16x8 a, u16x8 b, f32x4 c) {
    if constexpr (std::is_same<T, BF16>::value)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 scores(Chunk k, Chunk q, f32x4 c) { return mfma(k.x, q.x, c); }
  // the weights of a lane's 8 keys as an operand, and the product with their values' element e
  struct Weights {
    u16x8 x;
  };
  static __device__ __forceinline__ Weights weights(const float (&y)[8]) {
    const u32x4 w = {T::pack2(y[0], y[1]), T::pack2(y[2], y[3]), T::pack2(y[4], y[5]), T::pack2(y[6], y[7])};
    return Weights{__builtin_bit_cast(u16x8, w)};
  }
  static __device__ __forceinline__ f32x4 sums(const Values (&v)[8], int e, const Weights& w, f32x4 c) {
    u16x8 a;
#pragma unroll
    for (int j = 0; j < 8; j++) a[j] = v[j].x[e];
    return mfma(a, w.x, c);
  }
};
template <int W>
struct Operands<F32, W> {
  typedef float S;
  static constexpr int PER = 4;
  struct Chunk {
    f32x4 x;
  };
  struct Values {
    float x[W];
  };
  static __device__ __forceinline__ f32x4 scores(Chunk k, Chunk q, f32x4 c) {
#pragma unroll
    for (int t = 0; t < 4; t++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(k.x[t], q.x[t], c, 0, 0, 0);
    return c;
  }
  struct Weights {
    float x[8];
  };
  static __device__ __forceinline__ Weights weights(const float (&y)[8]) {
    Weights w;
#pragma unroll
    for (int j = 0; j < 8; j++) w.x[j] = y[j];
    return w;
  }
  static __device__ __forceinline__ f32x4 sums(const Values (&v)[8], int e, const Weights& w, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j].x[e], w.x[j], c, 0, 0, 0);
    return c;
  }
};

template <typename T, int D, int NR, int waves, int blocks>
__global__ __launch_bounds__(64 * waves, blocks) void paged_token(PagedFast a, PagedView v) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr int W = D / 16;
  typedef Operands<T, W> O;
  typedef typename O::S S;
  constexpr int PER = O::PER, KS = D / (4 * PER), R = 16 * NR;
  __shared__ float lds[waves * 16 * 17 + waves * NR * 32];
  __shared__ int found;  // values that are not finite were taken out
  constexpr float UP = std::is_same<T, F16>::value ? 7.f : 0.f;  // float16 weights times 2^7: see shift_of in attend_mfma.h
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  int id = blockIdx.x;
  const int kvh = id % v.kv_heads;
  id /= v.kv_heads;
  const int part = id % a.parts, slot = id / a.parts;
  zero_idle(v, (S*)a.out, 64 * waves);
  const Item it = item_at(v, slot, R);
  if (!it.live) return;
  const Sequence& q = it.seq;
  const Rules r = paged_rules(v);
  const int group = v.group, rows = q.n * group, tile = it.tile;
  const S* fresh_k = a.k != nullptr ? (const S*)a.k + kvh * (int64_t)v.hd : nullptr;
  const S* fresh_v = a.k != nullptr ? (const S*)a.v + kvh * (int64_t)v.hd : nullptr;
  if (part == 0 && fresh_k != nullptr) put_rows<S, PER>(v, it.s, q, kvh, (tile * R + group - 1) / group, min(q.n, (tile * R + R + group - 1) / group), fresh_k, fresh_v, (S*)a.key_pages, (S*)a.value_pages, 64 * waves);

  // this lane's rows: packed row -> token, head
  int p[NR];
  float slope2[NR];
  int64_t at[NR];
  bool there[NR];
  typename O::Chunk qf[NR][KS];
  f32x4 acc[NR][W];
  float m[NR], l[NR];
#pragma unroll
  for (int t = 0; t < NR; t++) {
    const int row = tile * R + t * 16 + n;
    there[t] = row < rows;
    const int i = there[t] ? row / group : 0, head = kvh * group + (there[t] ? row - i * group : 0);
    p[t] = q.off + i;
    at[t] = (int64_t)(q.row0 + i) * v.heads + head;
    slope2[t] = v.slopes != nullptr ? v.slopes[head] * PAGED_LOG2E : 0.f;
    const S* from = (const S*)a.q + (q.row0 + i) * v.q_row + head * (int64_t)v.hd;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const int d = PER * (4 * s + g);
      qf[t][s] = *(const typename O::Chunk*)(there[t] && d < v.hd ? from + d : (const S*)paged_zeros);
    }
#pragma unroll
    for (int e = 0; e < W; e++) acc[t][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[t] = -__builtin_inff();
    l[t] = 0.f;
  }
  const int pmin = q.off + tile * R / group, pmax = q.off + (min(tile * R + R, rows) - 1) / group;

  const Span span = span_of(v, q, tile, R, fresh_k != nullptr, KEYS);
  const int held = span.held, end = span.end, old_tiles = span.old_tiles, tiles = span.tiles;
  const int first = part * a.part_tiles, last = min(tiles, first + a.part_tiles);
  if (part > 0 && first >= tiles) return;

  const S* pool_k = (const S*)a.key_pages;
  const S* pool_v = (const S*)a.value_pages;
  typename O::Chunk kr[2][KS];
  typename O::Values vr[8];
  // a tile: its keys from k0 on, up to k1; from the pages if it is an old one
  auto begin_of = [&](int kt) __attribute__((always_inline)) { return kt < old_tiles ? kt * KEYS : held + (kt - old_tiles) * KEYS; };
  // the place of key lane % 32 of a tile as a row of the pools, -1 where there is none: of new ones whether there is a place
  auto look_up = [&](int kt) __attribute__((always_inline)) {
    const int j = begin_of(kt) + (lane & 31), stop = kt < old_tiles ? held : end;
    unsigned row = 0xffffffffu;
    if (kt < last && j < stop) {
      const int t = v.div.quotient(j), page = v.table[(int64_t)it.s * v.table_pages + t];
      if ((unsigned)page < (unsigned)v.pages) row = ((unsigned)page * v.kv_heads + kvh) * v.div.page + (j - t * v.div.page);
    }
    return row;
  };
  auto load_k = [&](int kt, unsigned rows_) __attribute__((always_inline)) {
    const bool old = kt < old_tiles;
    const uint64_t base = (uint64_t)(old ? pool_k : fresh_k + (q.row0 + begin_of(kt) - q.off) * v.k_row) + 16 * g;
    const unsigned stride = (unsigned)(old ? v.hd : v.k_row) * (unsigned)sizeof(S);
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const unsigned row = __shfl((int)rows_, 16 * t + n);
      const uint64_t from = base + (uint64_t)(old ? row : (unsigned)(16 * t + n)) * stride;
#pragma unroll
      for (int s = 0; s < KS; s++) kr[t][s] = *(const typename O::Chunk*)or_zeros(row != 0xffffffffu && PER * (4 * s + g) < v.hd, from + 64 * s);
    }
  };
  auto load_v = [&](int kt, unsigned rows_) __attribute__((always_inline)) {
    const bool old = kt < old_tiles;
    const uint64_t base = (uint64_t)(old ? pool_v : fresh_v + (q.row0 + begin_of(kt) - q.off) * v.v_row) + sizeof(S) * value_dim(n, W, v.hd);
    const unsigned stride = (unsigned)(old ? v.hd : v.v_row) * (unsigned)sizeof(S);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int key = 16 * (j >> 2) + 4 * g + (j & 3);
      const unsigned row = __shfl((int)rows_, key);
      vr[j] = *(const typename O::Values*)or_zeros(row != 0xffffffffu && W * n < v.hd, base + (uint64_t)(old ? row : (unsigned)key) * stride);
    }
  };
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  int kt = first + wave;
  unsigned here = look_up(kt), next = look_up(kt + waves);
  if (kt < last) {
    load_k(kt, here);
    load_v(kt, here);
  }
  for (; kt < last; kt += waves) {
    const int k0 = begin_of(kt);
    const bool more = kt + waves < last, partial = k0 + KEYS - 1 > pmin;  // partial: rows of the tile may not see all of the keys
    const unsigned after = look_up(kt + 2 * waves);
    f32x4 s[NR][2];
#pragma unroll
    for (int t = 0; t < NR; t++)
#pragma unroll
      for (int c = 0; c < 2; c++) s[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int t = 0; t < NR; t++) s[t][c] = O::scores(kr[c][ks], qf[t][ks], s[t][c]);
    const unsigned good = (unsigned)__ballot(here != 0xffffffffu);  // of the tile's 32 keys, those that are there
    if (more) load_k(kt + waves, next);
    const bool edge = good != 0xffffffffu || partial;
    float y[NR][8];
#pragma unroll
    for (int t = 0; t < NR; t++) {
      float mx = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < 8; j++) y[t][j] = s[t][j >> 2][j & 3];
      if (r.cap_out > 0.f) {
        cap_scores<8>(y[t], r);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) y[t][j] *= r.c2;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int in = 16 * (j >> 2) + 4 * g + (j & 3);
        float x = fmaf(-slope2[t], (float)(p[t] - k0 - in), y[t][j]);
        if (edge) x = ((good >> in) & 1) && k0 + in <= p[t] ? x : -__builtin_inff();
        y[t][j] = x;
        mx = fmaxf(mx, x);
      }
      if (__any(mx > m[t] + 8.f)) {
        mx = col_max(mx);
        const float up = fmaxf(m[t], mx), alpha = up == -__builtin_inff() ? 1.f : fast_exp2(m[t] - up);
        l[t] *= alpha;
#pragma unroll
        for (int e = 0; e < W; e++) acc[t][e] *= alpha;
        m[t] = up;
      }
      const float base = (m[t] == -__builtin_inff() ? 0.f : m[t]) - UP;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        y[t][j] = fast_exp2(y[t][j] - base);
        l[t] += y[t][j];
      }
    }
    if (partial && pmin != pmax) {  // see give_back
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int e = 0; e < W; e++)
          if (is_odd<T>(vr[j].x[e])) {
            vr[j].x[e] = 0;
            found = 1;
          }
    }
#pragma unroll
    for (int t = 0; t < NR; t++) {
      const typename O::Weights w = O::weights(y[t]);
#pragma unroll
      for (int e = 0; e < W; e++) acc[t][e] = O::sums(vr, e, w, acc[t][e]);
    }
    if (more) load_v(kt + waves, next);
    here = next;
    next = after;
  }
  // join the waves in order, one 16-dim slice of one row tile at a time
  float* sm = lds + waves * 16 * 17;
#pragma unroll
  for (int t = 0; t < NR; t++) {
    l[t] = col_sum(l[t]);
    if (g == 0) {
      sm[(wave * NR + t) * 32 + n] = m[t];
      sm[(wave * NR + t) * 32 + 16 + n] = l[t];
    }
  }
  __syncthreads();
  const int64_t rows_all = (int64_t)v.tokens * v.heads;
#pragma unroll
  for (int t = 0; t < NR; t++) {
    float top = -__builtin_inff(), total = 0.f;
    for (int w = 0; w < waves; w++) top = fmaxf(top, sm[(w * NR + t) * 32 + n]);
    for (int w = 0; w < waves; w++) {
      const float mw = sm[(w * NR + t) * 32 + n], lw = sm[(w * NR + t) * 32 + 16 + n];
      total += mw == -__builtin_inff() ? lw : lw * fast_exp2(mw - top);
    }
    const float factor = m[t] == -__builtin_inff() ? 1.f : fast_exp2(m[t] - top);
    const bool alone = tiles <= a.part_tiles;  // the sequence has one part: no partial results
    if (!alone && wave == 0 && g == 0 && there[t]) {
      float* st = a.stats + (part * rows_all + at[t]) * 2;
      st[0] = top;
      st[1] = total;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int e = 0; e < W; e++) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; i++) lds[(wave * 16 + 4 * g + i) * 17 + n] = acc[t][e][i] * factor;  // the e-th dim of lane 4 g + i
      __syncthreads();
      if (wave < 4) {  // 16 dims x 16 rows: wave w takes dims 4 w + g of row n
        const int dd = 4 * wave + g, d = value_dim(dd, W, v.hd) + e;
        float x = 0.f;
        for (int w = 0; w < waves; w++) x += lds[(w * 16 + dd) * 17 + n];
        if (there[t] && W * dd < v.hd && d >= W * dd) {  // (a dim of the lane before is that one's to store)
          if (!alone)
            a.totals[(part * rows_all + at[t]) * v.hd + d] = x;
          else
            T::store((S*)a.out + at[t] * v.hd, d, total == 0.f ? 0.f : x * inv);
        }
      }
    }
    __syncthreads();
  }
  if (found != 0 && wave == 0)
    give_back<T>(v, it.s, q, kvh, begin_of(first), last == tiles ? end : begin_of(last), held, tile * R, min(tile * R + R, rows), fresh_v, pool_v,
                 (S*)a.out, tiles <= a.part_tiles ? nullptr : a.totals + part * rows_all * v.hd);
#endif
}

// Waves of a workgroup that has a row tile to itself: as many as its registers allow without spills.
template <typename T, int D, int NR>
constexpr int LONE_WAVES = std::is_same<T, F32>::value ? (D == 64 && NR == 1 ? 8 : 4) : (D == 64 && NR == 1 ? 16 : 8);
// Workgroups of 4 waves that share a CU. Two wide float32 row tiles (2 x 8 tokens, up to 4000 positions, 55 us with two, 37 with one)
// and a workgroup that is alone anyway (8 x 2000 positions of 128 dims 79 and 68) spill in half of the registers; one row tile
// spills less than a second workgroup gives (32 x 8192 positions 326 and 342).
template <typename T, int D, int NR>
constexpr int SHARING = std::is_same<T, F32>::value && D == 128 && NR == 2 ? 1 : 2;

template <typename T, int D, int NR>
int launch_token(const PagedArgs& a, const PagedFast& f, bool lone) {
  const PagedView v = paged_view(a);
  const int64_t blocks = paged_slots(a, 16 * NR) * a.kv_heads * f.parts;
  constexpr int LONE = LONE_WAVES<T, D, NR>;
  if (!one_launch(blocks, lone ? 64 * LONE : 256)) return fail(LIMN_HIP_EUNSUPPORTED, "attend_paged: sizes out of range, %lld workgroups exceed one launch", (long long)blocks);
  if (lone)
    hipLaunchKernelGGL((paged_token<T, D, NR, LONE, 1>), dim3((unsigned)blocks), dim3(64 * LONE), 0, a.stream, f, v);
  else
    hipLaunchKernelGGL((paged_token<T, D, NR, 4, SHARING<T, D, NR>>), dim3((unsigned)blocks), dim3(256), 0, a.stream, f, v);
  return check_hip(hipGetLastError(), "launching attention of few tokens over a paged cache");
}

template <typename T>
int launch_token_type(const PagedArgs& a, const PagedFast& f, bool lone) {
  if (token_width(a.hd) == 64) return f.rows == 16 ? launch_token<T, 64, 1>(a, f, lone) : launch_token<T, 64, 2>(a, f, lone);
  return f.rows == 16 ? launch_token<T, 128, 1>(a, f, lone) : launch_token<T, 128, 2>(a, f, lone);
}

}  // namespace

int launch_paged_token(const PagedArgs& a, const PagedFast& f, bool lone) {
  return a.dtype == LIMN_HIP_FLOAT32 ? launch_token_type<F32>(a, f, lone) : a.dtype == LIMN_HIP_FLOAT16 ? launch_token_type<F16>(a, f, lone) : launch_token_type<BF16>(a, f, lone);
}

}  // namespace limn
