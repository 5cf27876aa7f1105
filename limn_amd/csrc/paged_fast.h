// Shared by the kernels of attention over a paged cache that take the tokens of a sequence in tiles (paged_token.hip,
// paged_tiles.h): which tile a workgroup has, the score rules, the write of the new tokens, partial results.
#pragma once

#include "attend_rules.h"
#include "paged.h"

#include <type_traits>

namespace limn {

struct PagedFast {
  const void* q;
  const void* k;
  const void* v;
  void* key_pages;
  void* value_pages;
  void* out;
  float* totals;  // of sequences with more than one part: (parts, tokens * heads, hd)
  float* stats;   // (parts, tokens * heads, 2): the reference point of the exponentials in log2, and their sum
  int parts, part_tiles;  // parts at most; key tiles of a part
  int rows, keys;         // a row tile's packed rows, a key tile's keys
};

int launch_paged_token(const PagedArgs& a, const PagedFast& f, bool lone);  // lone: one workgroup of many waves a row tile
int launch_paged_tiles_64(const PagedArgs& a, const PagedFast& f);
int launch_paged_tiles_96(const PagedArgs& a, const PagedFast& f);
int launch_paged_tiles_128(const PagedArgs& a, const PagedFast& f);

// Slots for row tiles of `rows` packed rows: sequence s has those from starts[s] * group / rows + s on, one for every tile
// that it has and up to one more, so that a slot finds its sequence without a sum over those before it.
inline int64_t paged_slots(const PagedArgs& a, int rows) { return a.tokens * a.group() / rows + a.sequences; }

namespace {

constexpr float PAGED_LOG2E = ATT_LOG2E;
__device__ __attribute__((aligned(16))) const float paged_zeros[128] = {};  // what a lane reads of a key that is not there

// An address, or that of zeros where there is nothing. By masks: a choice of pointers becomes a branch for every load.
__device__ __forceinline__ uint64_t or_zeros(bool there, uint64_t at) {
  const uint64_t mask = (uint64_t)0 - (uint64_t)there;
  return (at & mask) | ((uint64_t)paged_zeros & ~mask);
}

// A tile of packed rows of one sequence.
struct Item {
  bool live;
  int s, tile;
  Sequence seq;
};

__device__ __forceinline__ int slot_of(const PagedView& v, int s, int rows) {
  return (int)((int64_t)min(max(v.starts[s], 0), v.tokens) * v.group / rows) + s;
}

// The tile of a slot: the last sequence whose slots begin at or before it.
__device__ __forceinline__ Item item_at(const PagedView& v, int slot, int rows) {
  Item it;
  it.s = last_sequence(v, slot, [&](int i) { return slot_of(v, i, rows); });
  it.tile = slot - slot_of(v, it.s, rows);
  it.seq = sequence_at(v, it.s);
  it.live = it.tile >= 0 && (int64_t)it.tile * rows < it.seq.n * v.group;
  return it;
}

// The key tiles, of `keys` keys, that a tile of rows has to visit: those of the keys in the pages, [0, held), then those of the
// new ones that some row of it sees, [held, end).
struct Span {
  int held, end, old_tiles, tiles;
};
__device__ __forceinline__ Span span_of(const PagedView& v, const Sequence& q, int tile, int rows, bool fresh, int keys) {
  const int last = q.off + (min(tile * rows + rows, q.n * v.group) - 1) / v.group;  // the last row's position
  Span x;
  x.end = min(q.len, max(last + 1, 0));
  x.held = fresh ? max(q.off, 0) : x.end;
  x.old_tiles = (x.held + keys - 1) / keys;
  x.tiles = x.old_tiles + (x.end - x.held + keys - 1) / keys;
  return x;
}

// Zeros to the rows of no sequence, over all workgroups of the launch.
template <typename S>
__device__ __forceinline__ void zero_idle(const PagedView& v, S* out, int threads) {
  const int before = min(max(v.starts[0], 0), v.tokens), behind = min(max(v.starts[v.sequences], before), v.tokens);
  const int idle = before + v.tokens - behind, elements = v.heads * v.hd;
  for (int r = blockIdx.x; r < idle; r += gridDim.x) {
    S* o = out + (int64_t)(r < before ? r : behind + r - before) * elements;
    for (int i = threadIdx.x; i < elements; i += threads) o[i] = S(0);
  }
}

// The keys and values of rows [i0, i1) of a sequence to their places, 16 bytes a thread.
template <typename S, int PER>
__device__ __forceinline__ void put_rows(const PagedView& v, int s, const Sequence& q, int kvh, int i0, int i1, const S* k, const S* val, S* key_pages, S* value_pages, int threads) {
  const int chunks = v.hd / PER, all = (i1 - i0) * chunks;
  for (int c = threadIdx.x; c < all; c += threads) {
    const int i = i0 + c / chunks, d = (c % chunks) * PER, p = q.off + i;
    if (p < 0) continue;
    const int64_t place = key_place(v, s, kvh, p);
    if (place < 0) continue;
    *(uint4*)(key_pages + place + d) = *(const uint4*)(k + (q.row0 + i) * v.k_row + d);
    *(uint4*)(value_pages + place + d) = *(const uint4*)(val + (q.row0 + i) * v.v_row + d);
  }
}

template <typename T>
__device__ __forceinline__ bool is_odd(typename T::Storage x) {  // an infinity or a NaN
  if constexpr (std::is_same<T, F32>::value)
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
  else
    return (x & (std::is_same<T, BF16>::value ? 0x7f80 : 0x7c00)) == (std::is_same<T, BF16>::value ? 0x7f80 : 0x7c00);
}

// A weight of 0 of a key that a row does not see, times a value that is not finite, would be NaN. So tiles of keys that some
// rows do not see have their values looked over; what is not finite there goes into the products as 0, and this adds it to
// the results as they are stored, for the rows that see it: an infinity or a NaN times any weight above 0 is itself, and the sum with it.
// One wave, for the keys [j0, j1) of a sequence and its packed rows [r0, r1), whose stores are done; to partial totals if
// `totals` is not nullptr.
template <typename T>
__device__ __forceinline__ void give_back(const PagedView& v, int s, const Sequence& q, int kvh, int j0, int j1, int held, int r0, int r1, const typename T::Storage* fresh,
                                          const typename T::Storage* pool, typename T::Storage* out, float* totals) {
  __threadfence_block();
  for (int j = j0; j < j1; j++) {
    const int64_t place = key_place(v, s, kvh, j);
    if (place < 0) continue;
    const typename T::Storage* from = j < held ? pool + place : fresh + (q.row0 + j - q.off) * v.v_row;
    for (int d = threadIdx.x & 63; d < v.hd; d += 64) {
      const typename T::Storage x = from[d];
      if (!is_odd<T>(x)) continue;
      for (int r = r0; r < r1; r++) {
        const int i = r / v.group;
        if (q.off + i < j) continue;
        const int64_t at = (((int64_t)(q.row0 + i) * v.heads + kvh * v.group + r - i * v.group)) * v.hd + d;
        if (totals != nullptr)
          totals[at] += T::load(&x, 0);
        else
          T::store(out, at, T::load(out, at) + T::load(&x, 0));
      }
    }
  }
}

// The score constants, as attend_rules.h has them.
__device__ __forceinline__ Rules paged_rules(const PagedView& v) {
  const RuleArgs a = {nullptr, nullptr, nullptr, nullptr, 0, 0, 1, v.scale, v.softcap};
  return rules_of(a, 0);
}

}  // namespace
}  // namespace limn
