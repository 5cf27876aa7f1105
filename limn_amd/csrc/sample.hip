// A token for each row of logits from a given uniform number (include/limn_hip.h, limn_hip_sample).
//
// With w_j = exp((x_j - max x) / temperature) and the order of x descending, equal ones by index, every filter keeps a
// beginning of the order, and so does the draw end one: each is a search for the place where a running count (top-k) or a
// running mass (top-p, the draw) passes a number. A row has a workgroup, which reads it
//  - for its largest logit;
//  - into a histogram of 2048 bins of equal width in (max - x) / temperature (of counts alone, if there is a top-k);
//  - for the members of the bins that matter, which it sorts: with a top-k those of all bins up to the border's, and everything
//    else is done on them; with a top-p that of its border and the ones that the draw can end in; or the draw's alone.
// Rows of up to 1024 logits are sorted whole. A bin with more than 1024 members (rows of equal logits) is taken apart by the bits
// of x instead, 11, 11 and 10 at a time.
//
// A few long rows are split over workgroups, a launch for each of the three readings (sample_largest, sample_spread,
// sample_members) and a last one that sorts and draws; what they pass on lies in the workspace. Whole numbers make the parts' sums
// the row's, in any order.
//
// What bounds it: 256 rows of 131072 float32 logits, a workgroup a CU, take 130 us: 19 for the largest (the 134 MB come once from
// memory and then from the last cache), 48 for the masses, which is the rate of 64-bit atomics on shared memory (48 cycles for 64
// of them), 24 for the members, 20 for sorting and placing. 64 rows of 65536 bfloat16 with a top-k take 28 us, one row of 50257 28
// in four launches of 3, 7, 9 and 9, chains of small steps; 32 rows of 256 9. (Tried for a top-k and no faster: the kth of every four threads' largest as a bound
// in place of the counts, 28 us.)
//
// Masses are whole numbers, w 2^F rounded with F such that a row's sum stays below 2^63: sums of them do not depend on
// the order that atomics come in, and they are exact to V 2^-F of the largest weight (2^-28 of it for 2^17 tokens at
// worst, 2^-37 as roundings go), where borders between tokens lie some 2^-17 apart. Weights are computed in 64 bits for
// the same reason: a border that is off by 2^-24 gives another token in one row of a hundred.

#include "common.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace limn {
namespace {

constexpr int BINS = 2048;
constexpr int PAD = 16;  // room behind a list

struct SampleArgs {
  const float* uniforms;
  const float* temperature;  // these four nullptr for none
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int* tokens;
  float* logprobs;  // or nullptr
  int64_t rows, vocab, row_stride;
  int bits;  // F
};

// x as an unsigned number of the same order: NaN as minus infinity, both zeros alike
__device__ __forceinline__ float cleaned(float x) { return x != x ? -__builtin_inff() : x + 0.f; }
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(cleaned(x));
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

constexpr unsigned NOTHING = 0x007fffffu;  // the key of minus infinity

// The first elements of the order: those with a larger key, and of those with this one the ones up to an index or, where it is not
// known (-1), `taken` of them; and their mass. Borders with the same key are found the same way.
struct Border {
  unsigned key, taken;
  int index;
  uint64_t mass;
};
__device__ __forceinline__ bool shorter(const Border& a, const Border& b) {
  return a.key > b.key || (a.key == b.key && (a.index >= 0 ? a.index < b.index : a.taken < b.taken));
}

template <int TH>
struct Shared {
  alignas(16) uint64_t list[TH + PAD];  // of elements, see Row::append
  uint64_t sums[TH / 64];
  unsigned counts[TH / 64];
  uint64_t found_mass, found_element;
  unsigned found_bin, found_count, listed, word;
  double powers[64];  // 2^(F + i / 64)
};
// The logits of three bins: a border's, and the draw's two (the second one empty where they are the same).
struct Three {
  float least[3], most[3];
  __device__ __forceinline__ bool has(int j, float v) const { return v >= least[j] && v <= most[j]; }
};
template <int TH>
struct Bins {
  uint64_t mass0[BINS], mass[BINS];
  unsigned count0[BINS], count[BINS];  // count0: where a top-k asks for it
  alignas(16) uint64_t list[3][TH + PAD];
  unsigned listed[3];
  Three at;
};
struct Nothing {};

// What a row over several workgroups keeps between its launches.
constexpr int LISTED = 1024, MOST_PARTS = 64;
struct SplitRow {
  uint64_t mass[BINS];         // of the histogram: masses, or counts where there is a top-k
  uint64_t lists[3][LISTED];   // elements of the border's bin and of the draw's two, or of all bins that a top-k keeps
  uint64_t m[3], total, kept;  // the masses before those bins; of all; of those that reach min_p
  unsigned listed[3];
  int found;  // whether the lists are of use
  float best[MOST_PARTS];
};

// What a search looks for: a number of elements, or a mass.
struct Target {
  bool counts;
  uint64_t least;
  __device__ __forceinline__ bool reached(uint64_t mass, unsigned count) const { return (counts ? (uint64_t)count : mass) >= least; }
};

// The first mass of a beginning that reaches p of the whole: the last one kept is the first with which it does; the first element
// always is kept.
__device__ __forceinline__ uint64_t least_mass(float p, uint64_t total) {
  const double want = ceil(fmax((double)p, 0.0) * (double)total);
  return want > 1.0 ? (uint64_t)want : 1;
}
// The mass before the drawn token, at most: u of the kept mass, and below the whole of it.
__device__ __forceinline__ uint64_t mass_before(float u, uint64_t total) {
  const double share = u > 0.f ? (double)u * (double)total : u == u ? 0.0 : (double)total;
  return share < (double)total ? min((uint64_t)share, total - 1) : total - 1;
}

// A row of logits, seen by a workgroup of TH threads.
template <typename T, int TH>
struct Row {
  typedef typename T::Storage S;
  static constexpr int PER = 16 / (int)sizeof(S), WAVES = TH / 64;
  const S* x;
  int vocab, bits, head, chunks;  // elements before the first 16-byte boundary, and whole 16-byte chunks from there
  float least, most;              // infinite logits have all of the mass: they go as the largest number, all others as minus infinity
  float top, inv;                 // the largest logit; 64 / temperature
  double top64, scale;            // 64 log2(e) / temperature
  Shared<TH>& sh;

  __device__ __forceinline__ Row(const S* x_, int vocab_, int bits_, Shared<TH>& sh_) : x(x_), vocab(vocab_), bits(bits_), least(-__builtin_inff()), most(__builtin_inff()), top(0.f), inv(0.f), top64(0.0), scale(0.0), sh(sh_) {
    head = min(vocab, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(S));
    chunks = (vocab - head) / PER;
  }

  __device__ __forceinline__ void set(float best, float t) {
    if (best == __builtin_inff()) {
      least = best;
      most = best = __FLT_MAX__;
    }
    top = best;
    top64 = (double)top;
    inv = 64.f / t;
    scale = 64.0 * 1.4426950408889634 / (double)t;
  }

  __device__ __forceinline__ float seen(float v) const { return v >= least ? fminf(v, most) : -__builtin_inff(); }

  // f(logit, index) for every element, some of them by this thread; WHOLE: one at most
  template <bool WHOLE = false, typename F>
  __device__ __forceinline__ void each(F f) const {
    if constexpr (WHOLE) {
      if ((int)threadIdx.x < vocab) f(seen(T::load(x, threadIdx.x)), (int)threadIdx.x);
      return;
    }
    const u32x4* body = (const u32x4*)(x + head);
    int c = threadIdx.x;
    constexpr int U = 4;
    for (; c + (U - 1) * TH < chunks; c += U * TH) {
      u32x4 w[U];
#pragma unroll
      for (int u = 0; u < U; u++) w[u] = body[c + u * TH];
      // four chunks on their way, one after another worked on by one copy of f's code: four copies' registers spilled
#pragma unroll 1
      for (int u = 0; u < U; u++) eight(u < 2 ? u == 0 ? w[0] : w[1] : u == 2 ? w[2] : w[3], head + (c + u * TH) * PER, f);
    }
    for (; c < chunks; c += TH) eight(body[c], head + c * PER, f);
    const int rest = vocab - chunks * PER;  // before and behind the chunks: fewer than 2 PER
    if ((int)threadIdx.x < rest) {
      const int i = (int)threadIdx.x < head ? (int)threadIdx.x : chunks * PER + (int)threadIdx.x;
      f(seen(T::load(x, i)), i);
    }
  }
  template <typename F>
  __device__ __forceinline__ void eight(u32x4 w, int i, F f) const {
#pragma unroll
    for (int e = 0; e < PER; e++) {
      if constexpr (PER == 4)
        f(seen(__uint_as_float(w[e])), i + e);
      else
        f(seen(T::unpack((u16)(w[e >> 1] >> (16 * (e & 1))))), i + e);
    }
  }

  // 64 log2 of v's weight, and no less than -70 * 64: such a weight rounds to 0
  __device__ __forceinline__ double exponent(float v) const { return fmax(((double)v - top64) * scale, -4480.0); }
  // 2^F exp((v - top) / temperature): 2^(x / 64) with x = k + r, |r| <= 1/2, is 2^(k / 64) from the table times the series of 2^(r / 64),
  // whose first term left out is below 2^-54.
  __device__ __forceinline__ double weight(double x) const {
    const double k = rint(x), r = x - k;
    double p = fma(r, 1.2417843701716923e-12, 5.732851688640402e-10);
    p = fma(p, r, 2.1173137155464774e-7);
    p = fma(p, r, 5.864904955056169e-5);
    p = fma(p, r, 1.0830424696249145e-2);
    p = fma(p, r, 1.0);
    const int n = (int)k;
    const uint64_t w = (uint64_t)__double_as_longlong(p * sh.powers[n & 63]);
    return __longlong_as_double((long long)(w + ((uint64_t)(unsigned)((n & ~63) << 14) << 32)));  // 2^(n / 64)'s whole part onto the exponent
  }
  // rounded: the sum with 2^52 has no bits below 1 (a weight is at most 2^52)
  __device__ __forceinline__ uint64_t whole64(double w) const { return (uint64_t)__double_as_longlong(w + 4503599627370496.0) - 0x4330000000000000ull; }
  __device__ __forceinline__ uint64_t whole(float v) const { return whole64(weight(exponent(v))); }
  // 64 bins an e-fold of the weight; monotone in v: each step rounds, none turns the order round
  __device__ __forceinline__ int bin(float v) const { return v == top ? 0 : (int)fminf((top - v) * inv, (float)(BINS - 1)); }

  template <bool WHOLE = false>
  __device__ __forceinline__ float largest_of() const {
    float best = -__builtin_inff();
    each<WHOLE>([&](float v, int) __attribute__((always_inline)) { best = fmaxf(best, v); });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor(best, o));
    if ((threadIdx.x & 63) == 0) sh.counts[threadIdx.x >> 6] = __float_as_uint(best);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) best = fmaxf(best, __uint_as_float(sh.counts[w]));
    __syncthreads();
    return best;
  }

  __device__ __forceinline__ uint64_t sum(uint64_t v) const {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.sums[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) v += sh.sums[w];
    __syncthreads();
    return v;
  }

  // m and c: of this thread's elements; what the threads before it have, and before all of them the given, comes back in bm and bc
  __device__ __forceinline__ void before(uint64_t m, unsigned c, uint64_t& bm, unsigned& bc) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t im = m;
    unsigned ic = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t um = __shfl_up((unsigned long long)im, o);
      const unsigned uc = __shfl_up(ic, o);
      if (lane >= o) {
        im += um;
        ic += uc;
      }
    }
    if (lane == 63) {
      sh.sums[wave] = im;
      sh.counts[wave] = ic;
    }
    __syncthreads();
    bm += im - m;
    bc += ic - c;
#pragma unroll
    for (int w = 0; w < WAVES; w++)
      if (w < wave) {
        bm += sh.sums[w];
        bc += sh.counts[w];
      }
    __syncthreads();
  }

  // The first bin at which everything up to and with it reaches the target; the mass and count before it
  // are added to m and c. Every thread gets it; BINS if there is none.
  __device__ __forceinline__ int first_bin(const uint64_t* mass, const unsigned* count, Target target, uint64_t& m, unsigned& c) const {
    constexpr int PT = BINS / TH;
    uint64_t pm = 0, bm = m;
    unsigned pc = 0, bc = c;
#pragma unroll
    for (int i = 0; i < PT; i++) {
      pm += mass[threadIdx.x * PT + i];
      pc += count[threadIdx.x * PT + i];
    }
    if (threadIdx.x == 0) sh.found_bin = BINS;
    before(pm, pc, bm, bc);
    if (!target.reached(bm, bc) && target.reached(bm + pm, bc + pc)) {  // one thread at most: both grow along the bins
      int i = 0;
      for (; i + 1 < PT; i++) {
        const uint64_t nm = bm + mass[threadIdx.x * PT + i];
        const unsigned nc = bc + count[threadIdx.x * PT + i];
        if (target.reached(nm, nc)) break;
        bm = nm;
        bc = nc;
      }
      sh.found_bin = threadIdx.x * PT + i;
      sh.found_mass = bm;
      sh.found_count = bc;
    }
    __syncthreads();
    const int b = sh.found_bin;
    if (b < BINS) {
      m = sh.found_mass;
      c = sh.found_count;
    }
    __syncthreads();
    return b;
  }

  // The same for a mass alone, where the sums along the bins are at hand: bm before this thread's two, m0 in the first of them.
  __device__ __forceinline__ int bin_at(uint64_t bm, uint64_t m0, uint64_t m1, uint64_t least, uint64_t& m) const {
    if (bm < least && least <= bm + m0 + m1) {  // one thread
      const bool second = bm + m0 < least;
      sh.found_bin = threadIdx.x * 2 + second;
      sh.found_mass = second ? bm + m0 : bm;
    }
    __syncthreads();
    const int b = sh.found_bin;
    m = sh.found_mass;
    __syncthreads();
    return b;
  }

  // The masses into the bins, what reaches least_weight summed in kept; of the last bin, which may have most of the elements, in
  // registers.
  __device__ __forceinline__ void masses(uint64_t* mass, bool some, double least_weight, uint64_t& kept) const {
    uint64_t rest = 0;
    each([&](float v, int) __attribute__((always_inline)) {
      const double w = weight(exponent(v));
      const uint64_t m = whole64(w);
      const int b = bin(v);
      if (some) kept += w >= least_weight ? m : 0;
      if (b < BINS - 1)
        atomicAdd((unsigned long long*)&mass[b], (unsigned long long)m);
      else
        rest += m;
    });
    rest = sum(rest);
    if (threadIdx.x == 0) mass[BINS - 1] = rest;
    __syncthreads();
  }

  __device__ __forceinline__ void clear(uint64_t* mass, unsigned* count) const {
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += TH) {
      mass[b] = 0;
      count[b] = 0;
    }
    __syncthreads();
  }

  // The least logit of bin b or a bin before it: 64 keys between the ones that are known are looked at at a time, by every wave.
  __device__ __forceinline__ float edge(int b) const {
    unsigned lo = NOTHING, hi = key_of(top);  // bin(of_key(hi)) <= b
    while (lo < hi) {
      const unsigned step = (hi - lo) / 64 + 1, lane = threadIdx.x & 63;
      auto probe = [&](unsigned l) __attribute__((always_inline)) { return hi - min(hi - lo, step * (l + 1)); };
      const uint64_t bad = ~__ballot(bin(of_key(probe(lane))) <= b);  // lanes from some one on
      const unsigned good = bad == 0 ? 64u : (unsigned)__builtin_ctzll(bad);
      const unsigned least = good == 0 ? hi : probe(good - 1);
      lo = bad == 0 ? least : probe(good) + 1;
      hi = least;
    }
    return of_key(hi);
  }

  // The bins of a top-p's border and of the draw's ends, whatever the border's place in its bin, and the masses before them, from
  // this thread's two of the histogram `mass`. Whether no bin between the draw's two has a mass.
  __device__ __forceinline__ bool windows(const uint64_t (&two)[2], const uint64_t* mass, uint64_t total, uint64_t kept, float p, float u, Three& at, uint64_t (&m)[3]) const {
    uint64_t bm = 0;
    unsigned c = 0;
    before(two[0] + two[1], 0u, bm, c);
    int b[3] = {-1, 0, 0};
    uint64_t lo = min(total, kept), hi = lo;
    if (p < 1.f) {
      b[0] = bin_at(bm, two[0], two[1], least_mass(p, total), m[0]);
      lo = min(m[0] + 1, kept);
      hi = min(m[0] + mass[b[0]], kept);
    }
    b[1] = bin_at(bm, two[0], two[1], mass_before(u, lo) + 1, m[1]);
    b[2] = bin_at(bm, two[0], two[1], mass_before(u, hi) + 1, m[2]);
    const bool same = b[1] == b[2], next = same || m[1] + mass[b[1]] == m[2];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave < 6) {  // each edge by a wave of its own
      const int j = wave >> 1, mine = j == 0 ? b[0] : j == 1 ? b[1] : b[2];
      const bool upper = wave & 1, none = j == 0 ? !(p < 1.f) : j == 2 && same;
      float x = upper ? -__builtin_inff() : __builtin_inff();
      if (!none) x = upper && mine == 0 ? __builtin_inff() : edge(mine - upper);
      if (!none && upper && mine > 0) x = of_key(key_of(x) - 1);
      if ((threadIdx.x & 63) == 0) (upper ? at.most : at.least)[j] = x;
    }
    if (same) m[2] = ~0ull;  // nothing lies behind it
    __syncthreads();
    return next;
  }

  // ... and the largest of bin b
  __device__ __forceinline__ float largest(int b) const { return b == 0 ? __builtin_inff() : of_key(key_of(edge(b - 1)) - 1); }

  // list takes an element (a larger key first, as the complement of its key above its index)
  __device__ __forceinline__ void append(uint64_t* list, unsigned& listed, float v, int i) const {
    const unsigned at = atomicAdd(&listed, 1u);
    if (at < TH) list[at] = ((uint64_t)~key_of(v) << 32) | (unsigned)i;
  }

  // The elements of the row that in(logit) is true of, in the order: each thread gets one as it is listed, or ~0. More than TH of
  // them: not all.
  template <typename F>
  __device__ __forceinline__ uint64_t sorted(F in, bool& all) const {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    each([&](float v, int i) __attribute__((always_inline)) {
      if (in(v)) append(sh.list, sh.listed, v, i);
    });
    __syncthreads();
    all = sh.listed <= TH;
    return all ? arranged(sh.list, (int)sh.listed) : ~0ull;
  }

  // a list of n elements: each thread gets the one of its place, or ~0
  __device__ __forceinline__ uint64_t arranged(uint64_t* list, int n) const {
    uint64_t e = (int)threadIdx.x < n ? list[threadIdx.x] : ~0ull;
    const int wave0 = (int)(threadIdx.x & ~63u);
    if (n <= 512) {  // the place of each is the number of those before it: n reads that all lanes share; a sorting network of 36 steps took 6 us for 256
      if (threadIdx.x < PAD) list[n + threadIdx.x] = ~0ull;
      __syncthreads();
      int rank = 0;
      if (wave0 < n) {
        for (int j = 0; j < n; j += PAD) {
          ulonglong2 o[PAD / 2];
#pragma unroll
          for (int i = 0; i < PAD / 2; i++) o[i] = *(const ulonglong2*)(list + j + 2 * i);
#pragma unroll
          for (int i = 0; i < PAD / 2; i++) rank += (int)(o[i].x < e) + (int)(o[i].y < e);
        }
      }
      __syncthreads();
      if ((int)threadIdx.x < n) list[rank] = e;
      __syncthreads();
      e = (int)threadIdx.x < n ? list[threadIdx.x] : ~0ull;
    } else {
      for (int k = 2; k <= TH; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
          uint64_t o;
          if (j >= 64) {
            __syncthreads();
            list[threadIdx.x] = e;
            __syncthreads();
            o = list[threadIdx.x ^ j];
          } else {
            o = __shfl_xor((unsigned long long)e, j);
          }
          const bool low = (threadIdx.x & j) == 0, up = (threadIdx.x & k) == 0;
          if (low == up ? o < e : o > e) e = o;
        }
    }
    __syncthreads();
    return e;
  }

  // Of the sorted elements e, each with its mass w and the mass m and count c before it: the first one that reaches the target. Every
  // thread gets it.
  __device__ __forceinline__ Border place(uint64_t e, uint64_t w, Target target, uint64_t m, unsigned c) const {
    if (threadIdx.x == 0) sh.found_element = ~0ull;
    __syncthreads();
    if (e != ~0ull && !target.reached(m, c) && target.reached(m + w, c + 1)) {
      sh.found_element = e;
      sh.found_mass = m + w;
    }
    __syncthreads();
    const uint64_t f = sh.found_element;
    const Border b = f == ~0ull ? Border{0u, 0xffffffffu, 0x7fffffff, 0} : Border{~(unsigned)(f >> 32), 0u, (int)(unsigned)f, sh.found_mass};
    __syncthreads();
    return b;
  }

  // ... of a bin's, sorted, with the mass m and count c before it
  __device__ __forceinline__ Border reaches(uint64_t e, Target target, uint64_t m, unsigned c) const {
    const uint64_t w = e == ~0ull ? 0 : whole(of_key(~(unsigned)(e >> 32)));
    before(w, e == ~0ull ? 0u : 1u, m, c);
    return place(e, w, target, m, c);
  }

  // The shortest beginning of the order that reaches the target, from the histogram.
  __device__ __forceinline__ Border find(Bins<TH>& bins, Target target) const {
    uint64_t m = 0;
    unsigned c = 0;
    const int b0 = first_bin(bins.mass0, bins.count0, target, m, c);
    if (b0 == BINS) return Border{0u, 0xffffffffu, 0x7fffffff, 0};
    bool all;
    const float least = edge(b0), most = largest(b0);
    const uint64_t e = sorted([=](float v) __attribute__((always_inline)) { return v >= least && v <= most; }, all);
    if (all) return reaches(e, target, m, c);
    unsigned prefix = 0;
    for (int level = 0; level < 3; level++) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, width = level == 2 ? 10 : 11;
      clear(bins.mass, bins.count);
      each([&](float v, int) __attribute__((always_inline)) {
        const unsigned k = key_of(v);
        if (bin(v) != b0 || (level > 0 && (k >> (shift + width)) != prefix)) return;
        const int b = (1 << width) - 1 - (int)((k >> shift) & ((1u << width) - 1));  // larger keys first
        atomicAdd(&bins.count[b], 1u);
        atomicAdd((unsigned long long*)&bins.mass[b], (unsigned long long)whole(v));
      });
      __syncthreads();
      const int b = first_bin(bins.mass, bins.count, target, m, c);
      prefix = (prefix << width) | (unsigned)((1 << width) - 1 - b);
    }
    // equal ones, each of the same mass
    const uint64_t each_mass = whole(of_key(prefix));
    unsigned lo = 1, hi = bins.count[1023 - (prefix & 1023u)];
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2;
      if (target.reached(m + mid * each_mass, c + mid)) hi = mid; else lo = mid + 1;
    }
    return Border{prefix, lo, -1, m + lo * each_mass};
  }

  // the index of the nth element with this key
  __device__ __forceinline__ int index_of(unsigned key, unsigned nth) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned passed = 0;
    for (int i0 = 0; i0 < vocab; i0 += TH) {
      const int i = i0 + threadIdx.x;
      const bool hit = i < vocab && key_of(seen(T::load(x, i))) == key;
      const uint64_t hits = __ballot(hit);
      __syncthreads();
      if (lane == 0) sh.counts[wave] = (unsigned)__popcll(hits);
      __syncthreads();
      unsigned mine = passed, all = passed;
      for (int w = 0; w < WAVES; w++) {
        if (w < wave) mine += sh.counts[w];
        all += sh.counts[w];
      }
      if (hit && mine + (unsigned)__popcll(hits & ((1ull << lane) - 1)) + 1 == nth) sh.word = (unsigned)i;
      if (all >= nth) break;
      passed = all;
    }
    __syncthreads();
    return (int)sh.word;
  }
};

// the largest logit of a split row, for a whole wave
__device__ __forceinline__ float row_best(const SplitRow& s, int parts) {
  float best = (int)(threadIdx.x & 63) < parts ? s.best[threadIdx.x & 63] : -__builtin_inff();
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor(best, o));
  return best;
}

// WHOLE: rows of up to TH logits. SPLIT: the last launch of split rows.
template <typename T, int TH, bool WHOLE, bool SPLIT>
__global__ __launch_bounds__(TH) void sample_rows(const typename T::Storage* __restrict__ logits, SampleArgs a, const SplitRow* split, int parts) {
  __shared__ Shared<TH> sh;
  __shared__ std::conditional_t<WHOLE, Nothing, Bins<TH>> bins;
  const int64_t n = blockIdx.x;
  const int vocab = (int)a.vocab;
  const float t = a.temperature != nullptr ? a.temperature[n] : 1.f, p = a.top_p != nullptr ? a.top_p[n] : 1.f, q = a.min_p != nullptr ? a.min_p[n] : 0.f, u = a.uniforms[n];
  const int k = a.top_k != nullptr ? a.top_k[n] : 0;
  if (threadIdx.x < 64) sh.powers[threadIdx.x] = exp2(a.bits + threadIdx.x * 0.015625);
  Row<T, TH> row(logits + n * a.row_stride, vocab, a.bits, sh);
  const SplitRow* given = SPLIT ? split + n : nullptr;
  const float best = SPLIT ? row_best(*given, parts) : row.template largest_of<WHOLE>();
  auto give = [&](int token, float logprob) {
    if (threadIdx.x != 0) return;
    a.tokens[n] = token;
    if (a.logprobs != nullptr) a.logprobs[n] = logprob;
  };
  if (best == -__builtin_inff()) {  // no number above minus infinity
    give(-1, -__builtin_inff());
    return;
  }
  if (!(t > 0.f)) {
    if (threadIdx.x == 0) sh.word = 0xffffffffu;
    __syncthreads();
    unsigned first = 0xffffffffu;
    row.template each<WHOLE>([&](float v, int i) __attribute__((always_inline)) {
      if (v == best) first = min(first, (unsigned)i);
    });
    if (first != 0xffffffffu) atomicMin(&sh.word, first);
    __syncthreads();
    give((int)sh.word, 0.f);
    return;
  }
  row.set(best, t);

  const double one = ldexp(1.0, a.bits);  // the largest weight
  const bool few = k > 0 && k < vocab;
  // either all that is kept, sorted, or a histogram
  bool whole = WHOLE;
  const bool lists = SPLIT && given->found != 0 && max(given->listed[0], max(given->listed[1], given->listed[2])) <= LISTED;
  uint64_t e = ~0ull, total = 0, kept = 0;
  const double least_weight = (double)q * one;
  if constexpr (WHOLE) {
    row.template each<true>([&](float v, int i) __attribute__((always_inline)) { sh.list[i] = ((uint64_t)~key_of(v) << 32) | (unsigned)i; });
    __syncthreads();
    e = row.arranged(sh.list, vocab);
  } else {
    if (!lists) row.clear(bins.mass0, bins.count0);
    if (lists && few) {
      if (threadIdx.x < given->listed[0]) sh.list[threadIdx.x] = given->lists[0][threadIdx.x];
      __syncthreads();
      e = row.arranged(sh.list, (int)given->listed[0]);
      whole = true;
    } else if (few) {
      row.each([&](float v, int) __attribute__((always_inline)) { atomicAdd(&bins.count0[row.bin(v)], 1u); });
      __syncthreads();
      uint64_t m = 0;
      unsigned c = 0;
      const int last = row.first_bin(bins.mass0, bins.count0, Target{true, (uint64_t)k}, m, c);
      if (c + bins.count0[last] <= TH) {
        const float lo = row.edge(last);
        e = row.sorted([=](float v) __attribute__((always_inline)) { return v >= lo; }, whole);
      }
    }
    if (!whole && !lists && SPLIT && !few) {  // the lists did not hold what they have to: the histogram is there
      for (int b = threadIdx.x; b < BINS; b += TH) {
        bins.mass0[b] = given->mass[b];
        total += given->mass[b];
      }
      if (threadIdx.x == 0) kept = given->kept;
      __syncthreads();
    } else if (!whole && !lists) {
      row.masses(bins.mass0, q > 0.f, least_weight, kept);
      for (int b = threadIdx.x; b < BINS; b += TH) total += bins.mass0[b];
    }
  }
  uint64_t w = 0, m = 0;  // sorted: this thread's element's mass, and the mass before it
  if (whole) {
    const double x = e == ~0ull ? 0.0 : row.weight(row.exponent(of_key(~(unsigned)(e >> 32))));
    total = w = row.whole64(x);
    kept = threadIdx.x == 0 || x >= least_weight ? w : 0;
    unsigned c = 0;
    row.before(w, 0u, m, c);
  }
  total = lists && !few ? given->total : row.sum(total);
  kept = q > 1.f ? (uint64_t)1 << a.bits : !(q > 0.f) ? total : lists && !few ? given->kept : row.sum(kept);  // past 1: the first alone
  Border end = {0u, 0xffffffffu, 0x7fffffff, 0}, b;
  bool drawn = false;
  if constexpr (!WHOLE) {
    // The border of a top-p lies in one bin, and the draw, whatever the border's place in it, in one or in two others most often:
    // one reading for the members of all three, where one for each border took 16 us more for 256 rows of 131072.
    uint64_t ms[3] = {0, 0, 0};
    if (lists && !few) {
      ms[0] = given->m[0], ms[1] = given->m[1], ms[2] = given->m[2];
      drawn = true;
    } else if (!whole && !few && !SPLIT && p < 1.f) {
      const uint64_t two[2] = {bins.mass0[2 * threadIdx.x], bins.mass0[2 * threadIdx.x + 1]};
      if (row.windows(two, bins.mass0, total, kept, p, u, bins.at, ms)) {
        if (threadIdx.x < 3) bins.listed[threadIdx.x] = 0;
        __syncthreads();
        const Three at = bins.at;
        row.each([&](float v, int i) __attribute__((always_inline)) {
          const bool border = at.has(0, v), one = at.has(1, v), two = at.has(2, v);
          if (border | one | two) {
            if (border) row.append(bins.list[0], bins.listed[0], v, i);
            if (one | two) row.append(bins.list[1 + two], bins.listed[1 + two], v, i);
          }
        });
        __syncthreads();
        drawn = max(bins.listed[0], max(bins.listed[1], bins.listed[2])) <= TH;
      }
    }
    if (drawn) {
      Target target = {false, least_mass(p, total)};
#pragma unroll 1
      for (int j = p < 1.f ? 0 : 3;;) {  // the border's list, then one of the draw's
        if (j == 3) {
          total = min(total, kept);
          target.least = mass_before(u, total) + 1;
          j = target.least > ms[2] ? 2 : 1;
        }
        uint64_t* list = bins.list[j];
        int listed = (int)(lists ? given->listed[j] : bins.listed[j]);
        if (lists && (int)threadIdx.x < listed) list[threadIdx.x] = given->lists[j][threadIdx.x];
        __syncthreads();
        b = row.reaches(row.arranged(list, listed), target, ms[j], 0);
        if (j > 0) break;
        total = b.mass;
        j = 3;
      }
    }
  }
  // top-k, top-p, and with all that is kept known, the draw
  for (int step = drawn ? 3 : few ? 0 : p < 1.f ? 1 : 2; step < 3; step++) {
    if (step == 1 && !(p < 1.f)) continue;
    if (step == 2) total = min(total, kept);
    const Target target = {step == 0, step == 0 ? (uint64_t)k : step == 1 ? least_mass(p, total) : mass_before(u, total) + 1};
    if constexpr (WHOLE) {
      b = row.place(e, w, target, m, threadIdx.x);
    } else {
      b = whole ? row.place(e, w, target, m, threadIdx.x) : row.find(bins, target);
    }
    if (step < 2 && shorter(b, end)) {
      end = b;
      total = b.mass;
    }
  }
  const int i = b.index >= 0 ? b.index : row.index_of(b.key, b.taken);
  give(i, (float)log(row.weight(row.exponent(of_key(b.key))) / (double)total));
}

// A split row's launches. A part's elements, and its row's settings.
template <typename T, int TH>
struct Part {
  int64_t n;
  int begin, count, k;
  float t, p, q, u;
  bool few;
  __device__ __forceinline__ Part(const SampleArgs& a, int each) {
    n = blockIdx.y;
    begin = min((int)a.vocab, (int)blockIdx.x * each);
    count = min((int)a.vocab - begin, each);
    t = a.temperature != nullptr ? a.temperature[n] : 1.f, p = a.top_p != nullptr ? a.top_p[n] : 1.f, q = a.min_p != nullptr ? a.min_p[n] : 0.f, u = a.uniforms[n];
    k = a.top_k != nullptr ? a.top_k[n] : 0;
    few = k > 0 && k < a.vocab;
  }
};

// The parts' largest logits; and the row's numbers cleared.
template <typename T, int TH>
__global__ __launch_bounds__(TH) void sample_largest(const typename T::Storage* __restrict__ logits, SampleArgs a, SplitRow* split, int each) {
  __shared__ Shared<TH> sh;
  const Part<T, TH> at(a, each);
  SplitRow& s = split[at.n];
  const Row<T, TH> row(logits + at.n * a.row_stride + at.begin, at.count, a.bits, sh);
  const float best = row.largest_of();
  if (threadIdx.x == 0) s.best[blockIdx.x] = best;
  for (int b = blockIdx.x * TH + threadIdx.x; b < BINS; b += gridDim.x * TH) s.mass[b] = 0;
  if (blockIdx.x == 0 && threadIdx.x < 3) s.listed[threadIdx.x] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) s.kept = 0;
}

// The histogram: of counts where there is a top-k.
template <typename T, int TH>
__global__ __launch_bounds__(TH) void sample_spread(const typename T::Storage* __restrict__ logits, SampleArgs a, SplitRow* split, int each) {
  __shared__ Shared<TH> sh;
  __shared__ uint64_t mass[BINS];
  const Part<T, TH> at(a, each);
  SplitRow& s = split[at.n];
  const float best = row_best(s, gridDim.x);
  if (best == -__builtin_inff() || !(at.t > 0.f)) return;
  if (threadIdx.x < 64) sh.powers[threadIdx.x] = exp2(a.bits + threadIdx.x * 0.015625);
  Row<T, TH> row(logits + at.n * a.row_stride + at.begin, at.count, a.bits, sh);
  row.set(best, at.t);
  for (int b = threadIdx.x; b < BINS; b += TH) mass[b] = 0;
  __syncthreads();
  if (at.few) {
    row.each([&](float v, int) __attribute__((always_inline)) { atomicAdd((unsigned long long*)&mass[row.bin(v)], 1ull); });
    __syncthreads();
  } else {
    uint64_t kept = 0;
    row.masses(mass, at.q > 0.f, (double)at.q * ldexp(1.0, a.bits), kept);
    if (at.q > 0.f) kept = row.sum(kept);
    if (threadIdx.x == 0 && kept != 0) atomicAdd((unsigned long long*)&s.kept, (unsigned long long)kept);
  }
  for (int b = threadIdx.x; b < BINS; b += TH)
    if (mass[b] != 0) atomicAdd((unsigned long long*)&s.mass[b], (unsigned long long)mass[b]);
}

// The members of the bins that matter. Every part finds those bins for itself.
template <typename T, int TH>
__global__ __launch_bounds__(TH) void sample_members(const typename T::Storage* __restrict__ logits, SampleArgs a, SplitRow* split, int each) {
  __shared__ Shared<TH> sh;
  __shared__ Three three;
  __shared__ uint64_t lists[3][TH];  // of this part
  __shared__ unsigned listed[3], place[3];
  const Part<T, TH> at(a, each);
  SplitRow& s = split[at.n];
  const float best = row_best(s, gridDim.x);
  if (best == -__builtin_inff() || !(at.t > 0.f)) return;
  Row<T, TH> row(logits + at.n * a.row_stride + at.begin, at.count, a.bits, sh);
  row.set(best, at.t);
  const uint64_t two[2] = {s.mass[2 * threadIdx.x], s.mass[2 * threadIdx.x + 1]};
  uint64_t m[3] = {0, 0, 0}, total = 0, kept = 0;
  bool found;
  if (at.few) {
    uint64_t bm = 0;
    unsigned c = 0;
    row.before(two[0] + two[1], 0u, bm, c);
    const int last = row.bin_at(bm, two[0], two[1], (uint64_t)at.k, m[0]);
    found = m[0] + s.mass[last] <= LISTED;
    const float lo = row.edge(last);
    if (threadIdx.x < 3) {
      three.least[threadIdx.x] = threadIdx.x == 0 ? lo : __builtin_inff();
      three.most[threadIdx.x] = threadIdx.x == 0 ? __builtin_inff() : -__builtin_inff();
    }
    __syncthreads();
  } else {
    total = row.sum(two[0] + two[1]);
    kept = at.q > 1.f ? (uint64_t)1 << a.bits : at.q > 0.f ? s.kept : total;
    found = row.windows(two, s.mass, total, kept, at.p, at.u, three, m);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    s.found = found;
    s.total = total;
    for (int j = 0; j < 3; j++) s.m[j] = m[j];
  }
  if (!found) return;
  if (threadIdx.x < 3) listed[threadIdx.x] = 0;
  __syncthreads();
  const Three in = three;
  row.each([&](float v, int i) __attribute__((always_inline)) {
    const bool border = in.has(0, v), one = in.has(1, v), two = in.has(2, v);
    if (border | one | two) {
      if (border) row.append(lists[0], listed[0], v, at.begin + i);
      if (one | two) row.append(lists[1 + two], listed[1 + two], v, at.begin + i);
    }
  });
  __syncthreads();
  if (threadIdx.x < 3) place[threadIdx.x] = listed[threadIdx.x] > 0 ? atomicAdd(&s.listed[threadIdx.x], listed[threadIdx.x]) : 0;
  __syncthreads();
  for (int j = 0; j < 3; j++)  // past the end: not all of them fit, and the last launch takes the row from its beginning
    if (threadIdx.x < listed[j] && place[j] + threadIdx.x < LISTED) s.lists[j][place[j] + threadIdx.x] = lists[j][threadIdx.x];
}

// Parts of a row: some 4096 logits each, and a workgroup for each CU in all; from seven on. (One workgroup a row and parts, with a
// top-p and with a top-k: 1 x 16384 23 and 27 us, 18 and 24; 1 x 32000 36 and 27, 24 and 24; 1 x 131072 77 and 27, 40 and 25; 32 x 32000
// 41 and 33, 25 and 27; 32 x 131072 97 and 50, 41 and 31; 64 x 50257 53 and 75, 26 and 30.)
int parts_of(int64_t rows, int64_t vocab) {
  const int64_t n = std::min(std::min((int64_t)MOST_PARTS, 256 / rows), vocab / 4096);
  return n < 7 ? 1 : (int)n;
}

// of a row's workgroup
int threads_of(int64_t vocab) { return vocab <= 256 ? 256 : 1024; }

template <typename T>
int sample_of(const void* logits, const SampleArgs& a, SplitRow* split, hipStream_t stream) {
  typedef typename T::Storage S;
  const dim3 grid((unsigned)a.rows);
  if (const int parts = parts_of(a.rows, a.vocab); parts > 1) {
    const dim3 many((unsigned)parts, (unsigned)a.rows), block(1024);
    const int each = (int)(((a.vocab + parts - 1) / parts + 7) / 8 * 8);
    hipLaunchKernelGGL((sample_largest<T, 1024>), many, block, 0, stream, (const S*)logits, a, split, each);
    hipLaunchKernelGGL((sample_spread<T, 1024>), many, block, 0, stream, (const S*)logits, a, split, each);
    hipLaunchKernelGGL((sample_members<T, 1024>), many, block, 0, stream, (const S*)logits, a, split, each);
    hipLaunchKernelGGL((sample_rows<T, 1024, false, true>), grid, block, 0, stream, (const S*)logits, a, (const SplitRow*)split, parts);
    return check_hip(hipGetLastError(), "launching sampling");
  }
  if (threads_of(a.vocab) == 256)
    hipLaunchKernelGGL((sample_rows<T, 256, true, false>), grid, dim3(256), 0, stream, (const S*)logits, a, nullptr, 1);
  else if (a.vocab <= 1024)
    hipLaunchKernelGGL((sample_rows<T, 1024, true, false>), grid, dim3(1024), 0, stream, (const S*)logits, a, nullptr, 1);
  else
    hipLaunchKernelGGL((sample_rows<T, 1024, false, false>), grid, dim3(1024), 0, stream, (const S*)logits, a, nullptr, 1);
  return check_hip(hipGetLastError(), "launching sampling");
}

}  // namespace
}  // namespace limn

using namespace limn;

extern "C" int64_t limn_hip_sample_workspace(int dtype, int64_t rows, int64_t vocab) {
  return rows > 0 && vocab > 0 && parts_of(rows, vocab) > 1 ? rows * (int64_t)sizeof(SplitRow) : 0;
}

extern "C" int limn_hip_sample(const void* logits, const void* uniforms, const void* temperature, const void* top_k, const void* top_p, const void* min_p,
                               void* tokens, void* logprobs, int dtype, int64_t rows, int64_t vocab, int64_t row_stride, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  if (dtype != LIMN_HIP_FLOAT32 && dtype != LIMN_HIP_FLOAT16 && dtype != LIMN_HIP_BFLOAT16)
    return fail(LIMN_HIP_EUNSUPPORTED, "sample: takes float32, float16 or bfloat16, not dtype code %d", dtype);
  if (rows < 1 || vocab < 1) return fail(LIMN_HIP_EINVAL, "sample: sizes must be positive (rows %lld, vocab %lld)", (long long)rows, (long long)vocab);
  if (row_stride < vocab) return fail(LIMN_HIP_EINVAL, "sample: rows of %lld elements overlap at a stride of %lld", (long long)vocab, (long long)row_stride);
  if (logits == nullptr || uniforms == nullptr || tokens == nullptr) return fail(LIMN_HIP_EINVAL, "sample: null buffer");
  const uintptr_t size = dtype == LIMN_HIP_FLOAT32 ? 4 : 2;
  const uintptr_t words = (uintptr_t)uniforms | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)tokens | (uintptr_t)logprobs;
  if ((uintptr_t)logits % size != 0 || words % 4 != 0) return fail(LIMN_HIP_EINVAL, "sample: buffers must be aligned to their element size");
  if (workspace_bytes < 0) return fail(LIMN_HIP_EINVAL, "sample: negative workspace size");
  if (vocab > (1 << 24) || !one_launch(rows, threads_of(vocab))) return fail(LIMN_HIP_EUNSUPPORTED, "sample: sizes out of range");
  const int64_t need = limn_hip_sample_workspace(dtype, rows, vocab);
  if (need > 0 && (workspace == nullptr || (uintptr_t)workspace % 16 != 0 || workspace_bytes < need))
    return fail(LIMN_HIP_EINVAL, "sample: needs a workspace of %lld bytes, 16-byte aligned", (long long)need);
  int log2v = 0;
  while (((int64_t)1 << log2v) < vocab) log2v++;
  const SampleArgs a = {(const float*)uniforms, (const float*)temperature, (const int*)top_k, (const float*)top_p, (const float*)min_p, (int*)tokens,
                        (float*)logprobs, rows, vocab, row_stride, 62 - log2v < 52 ? 62 - log2v : 52};
  const hipStream_t s = (hipStream_t)stream;
  SplitRow* split = (SplitRow*)workspace;
  return dtype == LIMN_HIP_FLOAT32 ? sample_of<F32>(logits, a, split, s) : dtype == LIMN_HIP_FLOAT16 ? sample_of<F16>(logits, a, split, s) : sample_of<BF16>(logits, a, split, s);
}
