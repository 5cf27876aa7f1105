// Attention over a paged cache for sequences of many new tokens (parts of prompts), half widths of hd a multiple of 8 up to
// 128, run at a tile width D of 64, 96 or 128 (dims past hd are zeros).
//
// The loop is attend_fwd_wide's (attend_mfma.h): a workgroup of 4 waves has 128 resident rows, 32 a wave, one a lane pair; keys
// and values stream past in swizzled LDS tiles of 64, copied there by DMA while the tile before is multiplied, a tile's
// exponentials and its V product issued beside the next tile's scores. What a paged cache changes:
//  - a row is a token and one of the query heads that share the key head, so that the group's heads share every tile;
//  - a lane looks up the place of one key of 64 in the table, two tiles ahead, and the DMA's lanes get the places of the rows
//    that they copy from it: an address of 64 bits a lane, pages of any size. A key that is not there is copied from zeros;
//  - the keys held before come from the pages, the new ones from where the caller has them: the same launch puts those in
//    their places, and nothing has to wait for that;
//  - only a sequence's last tiles have keys that some rows do not see. There the values are looked over before they are
//    used: elements that are not finite (a weight of 0 times one is NaN) become 0, and go to the rows that see them at the end;
//  - calls with few row tiles cut the keys into parts, joined behind (paged_join).
#pragma once

#include "attend_mfma.h"
#include "paged_fast.h"

namespace limn {
namespace {

typedef __attribute__((address_space(1))) const void global_void;

// Where the operands of a swizzled 64 x 128 tile (SwzReads128) or 64 x 64 tile lie. The latter's rows are 128 bytes, two to the 64
// banks: chunk c of row r at c ^ f(r), f's bit 2 that of r >> 1 and its bits 0 and 1 those of r >> 3, so that the 8 rows of one
// parity that a row read serves together have 8 f, and 4 rows of a transposing read two bits 2 a parity.
template <int D>
struct PagedReads : SwzReads128 {
  static constexpr int RB = 256;
  static __device__ __forceinline__ int swizzle(int r) { return swz128(r); }
  __device__ __forceinline__ PagedReads(int lane) : SwzReads128(lane) {}
};
template <>
struct PagedReads<64> {
  static constexpr int RB = 128;
  static __device__ __forceinline__ int swizzle(int r) { return (((r >> 1) & 1) << 2) | ((r >> 3) & 3); }
  int row[4], tr[2][2];
  __device__ __forceinline__ PagedReads(int lane) {
    const int n = lane & 31, h = lane >> 5, g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int ds = 0; ds < 4; ds++) row[ds] = n * RB + (((2 * ds + h) ^ swizzle(n)) * 16);
#pragma unroll
    for (int dt = 0; dt < 2; dt++)
#pragma unroll
      for (int jj = 0; jj < 2; jj++) {
        const int r = 4 * h + 8 * jj + (i >> 2), col = dt * 32 + 16 * (g & 1) + 4 * (i & 3);
        tr[dt][jj] = r * RB + (((col >> 3) ^ swizzle(r)) * 16) + (col & 7) * 2;
      }
  }
  __device__ __forceinline__ u16x8 rows(const u16* tile, int sub, int ds) const { return *(const u16x8*)((const char*)tile + row[ds] + sub * 32 * RB); }
  // f differs by the bits 3 and 4 of a row: rows k0 + .. of k0 a multiple of 16 have those of k0 and of their own (jj)
  __device__ __forceinline__ u16x8 transposed(const u16* tile, int k0, int dt) const {
    const char* p = (const char*)tile + k0 * RB;
    const int turn = ((k0 >> 3) & 3) * 16;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p + (tr[dt][0] ^ turn)));
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p + (tr[dt][1] ^ turn)));
    return __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

template <typename T, int D, Cap CAP, bool BIAS>
__global__ __launch_bounds__(THREADS, 2) void paged_tiles(PagedFast a, PagedView v, int slots) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr bool RAW = CAP == CAP_NONE && !BIAS;
  typedef PagedReads<D> Reads;
  constexpr int KS = D / 16, DT = D / 32, RB = Reads::RB, RPI = 1024 / RB, PASSES = TILE * RB / 1024 / WAVES, CPR = RB / 16;
  constexpr float UP = shift_of<T>(7.f);
  constexpr int ELEMS = TILE * RB / 2;
  __shared__ __attribute__((aligned(1024))) u16 K0[ELEMS];
  __shared__ __attribute__((aligned(1024))) u16 K1[ELEMS];
  __shared__ __attribute__((aligned(1024))) u16 V0[ELEMS];
  __shared__ __attribute__((aligned(1024))) u16 V1[ELEMS];
  __shared__ int found;  // values that are not finite were taken out

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  int id = blockIdx.x;
  const int kvh = id % v.kv_heads;
  id /= v.kv_heads;
  const int part = id % a.parts, slot = slots - 1 - id / a.parts;  // the last rows of a sequence see the most keys: they go first
  zero_idle(v, (u16*)a.out, THREADS);
  const Item it = item_at(v, slot, ATT_ROWS);
  if (!it.live) return;
  const Sequence& q = it.seq;
  const Rules r = paged_rules(v);
  const int group = v.group, rows = q.n * group, tile = it.tile, hd = v.hd;
  const u16* fresh_k = a.k != nullptr ? (const u16*)a.k + kvh * (int64_t)hd : nullptr;
  const u16* fresh_v = a.k != nullptr ? (const u16*)a.v + kvh * (int64_t)hd : nullptr;
  if (part == 0 && fresh_k != nullptr)
    put_rows<u16, 8>(v, it.s, q, kvh, (tile * ATT_ROWS + group - 1) / group, min(q.n, (tile * ATT_ROWS + ATT_ROWS + group - 1) / group), fresh_k, fresh_v, (u16*)a.key_pages,
                     (u16*)a.value_pages, THREADS);
  const Span span = span_of(v, q, tile, ATT_ROWS, fresh_k != nullptr, TILE);
  const int first = part * a.part_tiles, last = min(span.tiles, first + a.part_tiles);
  if (part > 0 && first >= span.tiles) return;

  const int w0 = tile * ATT_ROWS + wave * 32, row = w0 + n;  // packed rows of the sequence and key head
  const bool there = row < rows, idle = w0 >= rows;  // a wave without rows copies and looks over its part of the tiles alone
  const int i = (there ? row : 0) / group, head = kvh * group + (there ? row - i * group : 0), p = q.off + i;
  const int64_t at = (int64_t)(q.row0 + i) * v.heads + head;
  const int p_wave = q.off + min(w0, rows - 1) / group, p_block = q.off + tile * ATT_ROWS / group;  // the first rows' positions
  const float slope2 = BIAS && v.slopes != nullptr ? v.slopes[head] * LOG2E : 0.f;
  u16x8 qf[KS];
  {
    const u16* from = (const u16*)a.q + (q.row0 + i) * v.q_row + head * (int64_t)hd;
#pragma unroll
    for (int ds = 0; ds < KS; ds++) qf[ds] = *(const u16x8*)(there && ds * 16 + 8 * h < hd ? from + ds * 16 + 8 * h : (const u16*)paged_zeros);
  }
  const Reads ad(lane);
  const float unit = RAW ? r.c2 : 1.f, lift = RESCALE_LOG2 / unit;
  const u16* pool_k = (const u16*)a.key_pages;
  const u16* pool_v = (const u16*)a.value_pages;

  auto begin_of = [&](int t) __attribute__((always_inline)) { return t < span.old_tiles ? t * TILE : span.held + (t - span.old_tiles) * TILE; };
  // the place of key `lane` of a tile as a row of the pools, -1 where there is none: of new ones, whether there is a place
  auto look_up = [&](int t) __attribute__((always_inline)) {
    const int j = begin_of(t) + lane, stop = t < span.old_tiles ? span.held : span.end;
    unsigned place = 0xffffffffu;
    if (t < last && j < stop) {
      const int e = v.div.quotient(j), page = v.table[(int64_t)it.s * v.table_pages + e];
      if ((unsigned)page < (unsigned)v.pages) place = ((unsigned)page * v.kv_heads + kvh) * v.div.page + (j - e * v.div.page);
    }
    return place;
  };
  auto copy = [&](u16* to, const u16* pool, const u16* fresh, int64_t fresh_row, int t, unsigned places) __attribute__((always_inline)) {
    const bool old = t < span.old_tiles;
    const uint64_t base = (uint64_t)(old ? pool : fresh + (q.row0 + begin_of(t) - q.off) * fresh_row);
    const unsigned stride = (unsigned)(old ? hd : fresh_row) * 2u;
    unsigned place[PASSES];
#pragma unroll
    for (int x = 0; x < PASSES; x++) place[x] = (unsigned)__shfl((int)places, (x * WAVES + wave) * RPI + lane / CPR);
#pragma unroll
    for (int x = 0; x < PASSES; x++) {
      const int kr = (x * WAVES + wave) * RPI + lane / CPR, c = (lane % CPR) ^ Reads::swizzle(kr);
      const uint64_t from = or_zeros(place[x] != 0xffffffffu && c * 8 < hd, base + (uint64_t)(old ? place[x] : (unsigned)kr) * stride + c * 16);
      __builtin_amdgcn_global_load_lds((global_void*)from, (lds_void*)((char*)to + (x * WAVES + wave) * 1024), 16, 0, 0);
    }
  };
  // this wave's rows of a tile of values that some rows of the block do not see whole, looked over (see give_back)
  auto look_over = [&](u16* tile_v, int t) __attribute__((always_inline)) {
    if (begin_of(t) + TILE - 1 <= p_block) return;
#pragma unroll
    for (int x = 0; x < PASSES; x++) {
      u16x8* mine = (u16x8*)((char*)tile_v + (x * WAVES + wave) * 1024) + lane;
      u16x8 e = *mine;
      bool bad = false;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const bool o = is_odd<T>(e[k]);
        bad |= o;
        if (o) e[k] = 0;
      }
      if (bad) {
        *mine = e;
        found = 1;
      }
    }
  };

  f32x16 acc[DT], s[2];
  float m = neg_inf(), l = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; dt++) acc[dt] = zero16();
  auto scores = [&](const u16* Kt, f32x16 (&o)[2]) __attribute__((always_inline)) {
    o[0] = zero16();
    o[1] = zero16();
#pragma unroll
    for (int ds = 0; ds < KS; ds++)
#pragma unroll
      for (int sub = 0; sub < 2; sub++) o[sub] = T::mfma32(ad.rows(Kt, sub, ds), qf[ds], o[sub]);
  };
  // a tile's scores bent and masked, and the reference point moved where they pass it by more than 2^8
  auto look = [&](f32x16 (&o)[2], int k0, uint64_t good) __attribute__((always_inline)) {
    const float near = (float)(p - k0 - 4 * h);
#pragma unroll
    for (int sub = 0; sub < 2; sub++) {
      if (CAP == CAP_EXACT) cap_scores<16>(o[sub], r);
      if (!RAW) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
          float unused;
          o[sub][e] = bend<CAP, BIAS, false>(o[sub][e], r, slope2, near - (float)(sub * 32 + 8 * (e >> 2) + (e & 3)), unused);
        }
      }
      if ((unsigned)(good >> (32 * sub)) != 0xffffffffu || k0 + sub * 32 + 31 > p_wave) {
        const unsigned mine = (unsigned)(good >> (32 * sub)) >> (4 * h);
        const int seen = p - k0 - sub * 32 - 4 * h;
#pragma unroll
        for (int e = 0; e < 16; e++) o[sub][e] = ((mine >> (8 * (e >> 2) + (e & 3))) & 1) && 8 * (e >> 2) + (e & 3) <= seen ? o[sub][e] : neg_inf();
      }
    }
    float mx = neg_inf();
#pragma unroll
    for (int sub = 0; sub < 2; sub++)
#pragma unroll
      for (int e = 0; e < 16; e++) mx = fmaxf(mx, o[sub][e]);
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
  auto pipe = [&](auto has_next, const u16* Kn, const u16* Vc, int t, uint64_t good) __attribute__((always_inline)) {
    if (idle) return;
    f32x16 sn[2];
    if (decltype(has_next)::value) scores(Kn, sn);
    const float base = (m == neg_inf() ? 0.f : m * unit) - UP;
    float rs = 0.f;
#pragma unroll
    for (int sub = 0; sub < 2; sub++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const float x = RAW ? fast_exp2(fmaf(s[sub][e], unit, -base)) : fast_exp2(s[sub][e] - base);
        s[sub][e] = x;
        rs += x;
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
      look(sn, begin_of(t + 1), good);
      s[0] = sn[0];
      s[1] = sn[1];
    }
  };
  const int count = last - first;
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  if (count > 0) {
    // tile it's K and V are in buffers it % 2; K goes two tiles ahead, V one, the table three
    int t = first;
    const unsigned place0 = look_up(t);
    unsigned place1 = look_up(t + 1), place2 = look_up(t + 2);
    copy(K0, pool_k, fresh_k, v.k_row, t, place0);
    copy(V0, pool_v, fresh_v, v.v_row, t, place0);
    copy(K1, pool_k, fresh_k, v.k_row, t + 1, place1);
    __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
    look_over(V0, t);
    __syncthreads();
    const uint64_t good0 = __ballot(place0 != 0xffffffffu);
    if (!idle) {
      scores(K0, s);
      look(s, begin_of(t), good0);
    }
    __syncthreads();  // every wave's reads of K buffer 0 are done before the third tile is copied there
    auto step = [&](const u16* Kn, const u16* Vc, u16* Kf, u16* Vf) __attribute__((always_inline)) {
      copy(Kf, pool_k, fresh_k, v.k_row, t + 2, place2);
      copy(Vf, pool_v, fresh_v, v.v_row, t + 1, place1);
      const uint64_t good = __ballot(place1 != 0xffffffffu);
      place1 = place2;
      place2 = look_up(t + 3);
      pipe(std::true_type{}, Kn, Vc, t, good);
      t++;
      __builtin_amdgcn_s_waitcnt(WAIT_VMEM);
      look_over(Vf, t);
      __syncthreads();
    };
    int done = 0;
    for (; done + 2 < count; done += 2) {
      step(K1, V0, K0, V1);
      step(K0, V1, K1, V0);
    }
    if (done + 1 < count) {
      step(K1, V0, K0, V1);
      pipe(std::false_type{}, K0, V1, t, 0);
    } else {
      pipe(std::false_type{}, K0, V0, t, 0);
    }
  }
  const float total = pair_sum(l);
  __syncthreads();  // the tile buffers become staging below
  // the keys of this part, for what was taken out of their values
  const int j0 = begin_of(first), j1 = last == span.tiles ? span.end : begin_of(last);
  const bool odd = found != 0;
  if (span.tiles > a.part_tiles) {
    const int64_t rows_all = (int64_t)v.tokens * v.heads;
    if (there) {
      float* o = a.totals + (part * rows_all + at) * hd;
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int d = dt * 32 + 8 * k + 4 * h;
          if (d < hd) *(f32x4*)(o + d) = f32x4{acc[dt][4 * k], acc[dt][4 * k + 1], acc[dt][4 * k + 2], acc[dt][4 * k + 3]};
        }
      if (h == 0) {
        a.stats[(part * rows_all + at) * 2] = m == neg_inf() ? m : m * unit;
        a.stats[(part * rows_all + at) * 2 + 1] = total;
      }
    }
    if (odd) give_back<T>(v, it.s, q, kvh, j0, j1, span.held, w0, min(w0 + 32, rows), fresh_v, pool_v, nullptr, a.totals + part * rows_all * hd);
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;  // a row that sees nothing is a row of zeros
  // through LDS, so that a store instruction writes whole rows
  constexpr int RS = D + 8, CH = D / 8;
  static_assert(32 * RS <= ELEMS, "a wave's rows fit a tile's buffer");
  u16* stage = wave == 0 ? K0 : wave == 1 ? K1 : wave == 2 ? V0 : V1;
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const u16x4 o = {T::pack(acc[dt][4 * k] * inv), T::pack(acc[dt][4 * k + 1] * inv), T::pack(acc[dt][4 * k + 2] * inv), T::pack(acc[dt][4 * k + 3] * inv)};
      *(u16x4*)(stage + n * RS + dt * 32 + 8 * k + 4 * h) = o;
    }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < 32 * CH / 64; j++) {
    const int sr = (j * 64 + lane) / CH, c = (j * 64 + lane) % CH, pr = w0 + sr;
    const u16x8 x = *(const u16x8*)(stage + sr * RS + c * 8);
    if (pr < rows && c * 8 < hd) {
      const int pi = pr / group;
      *(u16x8*)((u16*)a.out + ((int64_t)(q.row0 + pi) * v.heads + kvh * group + pr - pi * group) * hd + c * 8) = x;
    }
  }
  if (odd) give_back<T>(v, it.s, q, kvh, j0, j1, span.held, w0, min(w0 + 32, rows), fresh_v, pool_v, (u16*)a.out, nullptr);
#endif
}

template <typename T, int D, Cap CAP, bool BIAS>
int launch_tiles_as(const PagedArgs& a, const PagedFast& f) {
  const int64_t slots = paged_slots(a, ATT_ROWS), blocks = slots * a.kv_heads * f.parts;
  if (!one_launch(blocks, THREADS)) return fail(LIMN_HIP_EUNSUPPORTED, "attend_paged: sizes out of range, %lld workgroups exceed one launch", (long long)blocks);
  hipLaunchKernelGGL((paged_tiles<T, D, CAP, BIAS>), dim3((unsigned)blocks), dim3(THREADS), 0, a.stream, f, paged_view(a), (int)slots);
  return check_hip(hipGetLastError(), "launching attention over a paged cache");
}

template <typename T, int D>
int launch_tiles_rules(const PagedArgs& a, const PagedFast& f) {
  const bool bias = a.slopes != nullptr;
  if (a.softcap > CAP_SHORT_MOST) return launch_tiles_as<T, D, CAP_EXACT, true>(a, f);  // slopes of 0 without any
  if (a.softcap > 0) return bias ? launch_tiles_as<T, D, CAP_SHORT, true>(a, f) : launch_tiles_as<T, D, CAP_SHORT, false>(a, f);
  return bias ? launch_tiles_as<T, D, CAP_NONE, true>(a, f) : launch_tiles_as<T, D, CAP_NONE, false>(a, f);
}

}  // namespace
}  // namespace limn
