// Attention of packed new tokens over a paged cache (include/limn_hip.h, limn_hip_attend_paged): arguments, and how a kernel
// finds a sequence's rows and a key's place.
//
//   sequence s: rows [starts[s], starts[s + 1]) of q, k and v, n of them, its positions len - n .. len - 1;
//   key j of s: place j % page of page table[s, j / page] of (pages, kv_heads, page, hd);
//   s[i, j] = cap(scale q_i . k_j) - slope_h (p(i) - j),  seen: j <= p(i), a page inside the cache.
#pragma once

#include "common.h"

namespace limn {

// One call, already validated.
struct PagedArgs {
  const void* q;
  const void* k;  // nullptr, and v too: the cache holds the new tokens already
  const void* v;
  void* key_pages;
  void* value_pages;
  const int* starts;
  const int* lengths;
  const int* table;
  const float* slopes;  // (heads) or nullptr
  void* out;
  int dtype;
  int64_t tokens, sequences, heads, kv_heads, hd, pages, page, table_pages;
  int64_t q_row, k_row, v_row;  // elements between tokens
  double scale, softcap;
  void* workspace;
  int64_t workspace_bytes;
  hipStream_t stream;
  int group() const { return (int)(heads / kv_heads); }
};

// j / page for 0 <= j < 2^31 as a product: with b = ceil(log2 page) and m = floor(2^(31 + b) / page) + 1 < 2^32 the
// excess of j m / 2^(31 + b) over j / page is below j / 2^(31 + b) <= 1 / page, so its floor is exact.
struct PageDiv {
  unsigned mul, page;
  int shift;
  static PageDiv of(int64_t page) {
    int b = 0;
    while (((int64_t)1 << b) < page) b++;
    return PageDiv{(unsigned)((((uint64_t)1 << (31 + b)) / (uint64_t)page) + 1), (unsigned)page, 31 + b};
  }
  __host__ __device__ __forceinline__ int quotient(int j) const { return (int)(((uint64_t)(unsigned)j * mul) >> shift); }
};

// What the kernels take.
struct PagedView {
  const int* starts;
  const int* lengths;
  const int* table;
  const float* slopes;
  int tokens, sequences, heads, kv_heads, group, hd, pages, table_pages;
  int64_t q_row, k_row, v_row, page_elements;  // kv_heads * page * hd
  PageDiv div;
  float scale, softcap;
};

inline PagedView paged_view(const PagedArgs& a) {
  return PagedView{a.starts, a.lengths, a.table, a.slopes, (int)a.tokens, (int)a.sequences, (int)a.heads, (int)a.kv_heads, a.group(), (int)a.hd, (int)a.pages,
                   (int)a.table_pages, a.q_row, a.k_row, a.v_row, a.kv_heads * a.page * a.hd, PageDiv::of(a.page), (float)a.scale, (float)a.softcap};
}

// A sequence's rows and positions. Whatever the device's numbers are, rows stay inside the tokens and positions inside
// the table.
struct Sequence {
  int row0, n, len, off;  // off: the position of row 0, below 0 if there are more rows than positions
};
__device__ __forceinline__ Sequence sequence_at(const PagedView& v, int s) {
  const int b = min(max(v.starts[s], 0), v.tokens), e = min(max(v.starts[s + 1], b), v.tokens);
  const int len = (int)min((int64_t)max(v.lengths[s], 0), (int64_t)v.table_pages * v.div.page);
  return Sequence{b, e - b, len, len - (e - b)};
}

// The last sequence whose place(s), which does not fall along the sequences, is at most `at`; the first if there is none. For
// a whole wave at a time: 64 sequences are looked at with one load.
template <typename F>
__device__ __forceinline__ int last_sequence(const PagedView& v, int at, F place) {
  const int lane = threadIdx.x & 63;
  int lo = 0, span = v.sequences;
  while (span > 1) {
    const int step = (span + 63) / 64;
    const uint64_t before = __ballot(lane * step < span && place(min(lo + lane * step, v.sequences - 1)) <= at);
    const int k = before == 0 ? 0 : 63 - __builtin_clzll(before);
    lo += k * step;
    span = min(step, span - k * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The sequence of a row, or -1: the last one that starts at or before it, if it reaches the row. For a whole wave.
__device__ __forceinline__ int sequence_of(const PagedView& v, int row) {
  const int s = last_sequence(v, row, [&](int i) { return v.starts[i]; });
  return v.starts[s] <= row && row < v.starts[s + 1] ? s : -1;
}

// The elements before key j of sequence s and key head h in the pages, or -1 where its page is not one of the cache's.
__device__ __forceinline__ int64_t key_place(const PagedView& v, int s, int h, int j) {
  const int t = v.div.quotient(j), page = v.table[(int64_t)s * v.table_pages + t];
  if ((unsigned)page >= (unsigned)v.pages) return -1;
  return page * v.page_elements + ((int64_t)h * v.div.page + (j - t * (int)v.div.page)) * v.hd;
}

}  // namespace limn
