// A token for each row of logits from a given uniform number (include/limn_hip.h, limn_hip_sample).
//
// With w_j = exp((x_j - max x) / temperature) and the order of x descending, equal ones by index, every filter keeps a
// beginning of the order, and so does the draw end one: each is a search for the place where a running count (top-k) or a
// running mass (top-p, the draw) passes a number. A row's workgroup finds such a place by histograms: 2048 bins of equal
// width in (max - x) / temperature, then the key bits of x inside the bin that it lies in, 11, 11 and 10 at a time.
//
// Masses are whole numbers, w 2^F rounded with F such that a row's sum stays below 2^63: sums of them do not depend on
// the order that atomics come in, and they are exact to V 2^-F of the largest weight (2^-28 of it for 2^17 tokens at
// worst, 2^-37 as roundings go), where borders between tokens lie some 2^-17 apart. Weights are computed in 64 bits for
// the same reason: a border that is off by 2^-24 gives another token in one row of a hundred.

#include "common.h"

#include <math.h>

namespace limn {
namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64, BINS = 2048;

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
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x != x ? -__builtin_inff() : x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

constexpr unsigned NOTHING = 0x007fffffu;  // the key of minus infinity

// The first elements of the order: those with a larger key, and `taken` of those with this one.
struct Border {
  unsigned key, taken;
};
__device__ __forceinline__ bool shorter(Border a, Border b) { return a.key > b.key || (a.key == b.key && a.taken < b.taken); }

struct Shared {
  uint64_t mass0[BINS], mass[BINS], sums[WAVES];
  unsigned count0[BINS], count[BINS], counts[WAVES];
  uint64_t found_mass;
  unsigned found_bin, found_count, word;
};

template <typename T>
struct Row {
  const typename T::Storage* x;
  int vocab, bits;
  float top, inv;  // the largest logit; 1 / temperature
  double inv64;
  Shared& sh;

  __device__ __forceinline__ float at(int i) const { return T::load(x, i); }
  __device__ __forceinline__ double weight(float v) const { return v == top ? 1.0 : exp(((double)v - (double)top) * inv64); }
  __device__ __forceinline__ uint64_t whole(float v) const { return (uint64_t)rint(ldexp(weight(v), bits)); }
  // monotone in v: each step rounds, none turns the order round
  __device__ __forceinline__ int bin(float v) const { return v == top ? 0 : (int)fminf((top - v) * inv * 64.f, (float)(BINS - 1)); }

  __device__ uint64_t sum(uint64_t v) const {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.sums[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < WAVES; w++) v += sh.sums[w];
    return v;
  }

  __device__ void clear(uint64_t* mass, unsigned* count) const {
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += THREADS) {
      mass[b] = 0;
      count[b] = 0;
    }
    __syncthreads();
  }

  // The first bin at which reached(mass, count) of everything up to and with it is true; the mass and count before it
  // are added to m and c. Every thread gets it; BINS if there is none.
  template <typename F>
  __device__ int first_bin(const uint64_t* mass, const unsigned* count, F reached, uint64_t& m, unsigned& c) const {
    constexpr int PER = BINS / THREADS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t pm = 0;
    unsigned pc = 0;
    for (int i = 0; i < PER; i++) {
      pm += mass[threadIdx.x * PER + i];
      pc += count[threadIdx.x * PER + i];
    }
    uint64_t im = pm;
    unsigned ic = pc;
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t um = __shfl_up((unsigned long long)im, o);
      const unsigned uc = __shfl_up(ic, o);
      if (lane >= o) {
        im += um;
        ic += uc;
      }
    }
    if (threadIdx.x == 0) sh.found_bin = BINS;
    if (lane == 63) {
      sh.sums[wave] = im;
      sh.counts[wave] = ic;
    }
    __syncthreads();
    uint64_t bm = m + im - pm;
    unsigned bc = c + ic - pc;
    for (int w = 0; w < wave; w++) {
      bm += sh.sums[w];
      bc += sh.counts[w];
    }
    if (!reached(bm, bc) && reached(bm + pm, bc + pc)) {  // one thread at most: both grow along the bins
      int i = 0;
      for (; i + 1 < PER; i++) {
        const uint64_t nm = bm + mass[threadIdx.x * PER + i];
        const unsigned nc = bc + count[threadIdx.x * PER + i];
        if (reached(nm, nc)) break;
        bm = nm;
        bc = nc;
      }
      sh.found_bin = threadIdx.x * PER + i;
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

  // The shortest beginning of the order of which reached(mass, count) is true, or the whole of it: key 0.
  template <typename F>
  __device__ Border find(F reached) const {
    uint64_t m = 0;
    unsigned c = 0;
    const int b0 = first_bin(sh.mass0, sh.count0, reached, m, c);
    if (b0 == BINS) return Border{0u, 0xffffffffu};
    unsigned prefix = 0;
    for (int level = 0; level < 3; level++) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, width = level == 2 ? 10 : 11;
      clear(sh.mass, sh.count);
      for (int i = threadIdx.x; i < vocab; i += THREADS) {
        const float v = at(i);
        const unsigned k = key_of(v);
        if (bin(of_key(k)) != b0 || (level > 0 && (k >> (shift + width)) != prefix)) continue;
        const int b = (1 << width) - 1 - (int)((k >> shift) & ((1u << width) - 1));  // larger keys first
        atomicAdd(&sh.count[b], 1u);
        atomicAdd((unsigned long long*)&sh.mass[b], (unsigned long long)whole(of_key(k)));
      }
      __syncthreads();
      const int b = first_bin(sh.mass, sh.count, reached, m, c);
      prefix = (prefix << width) | (unsigned)((1 << width) - 1 - b);
    }
    // equal ones, each of the same mass
    const uint64_t each = whole(of_key(prefix));
    unsigned lo = 1, hi = sh.count[1023 - (prefix & 1023u)];
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2;
      if (reached(m + mid * each, c + mid)) hi = mid; else lo = mid + 1;
    }
    return Border{prefix, lo};
  }

  // the mass of a beginning of the order
  __device__ uint64_t mass_of(Border e) const {
    uint64_t v = 0;
    for (int i = threadIdx.x; i < vocab; i += THREADS) {
      const unsigned k = key_of(at(i));
      if (k > e.key) v += whole(of_key(k));
    }
    return sum(v) + (e.taken == 0xffffffffu ? 0 : e.taken * whole(of_key(e.key)));
  }

  // the index of the nth element with this key
  __device__ int index_of(unsigned key, unsigned nth) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned before = 0;
    for (int i0 = 0; i0 < vocab; i0 += THREADS) {
      const int i = i0 + threadIdx.x;
      const bool hit = i < vocab && key_of(at(i)) == key;
      const uint64_t hits = __ballot(hit);
      __syncthreads();
      if (lane == 0) sh.counts[wave] = (unsigned)__popcll(hits);
      __syncthreads();
      unsigned mine = before, all = before;
      for (int w = 0; w < WAVES; w++) {
        if (w < wave) mine += sh.counts[w];
        all += sh.counts[w];
      }
      if (hit && mine + (unsigned)__popcll(hits & ((1ull << lane) - 1)) + 1 == nth) sh.word = (unsigned)i;
      if (all >= nth) break;
      before = all;
    }
    __syncthreads();
    return (int)sh.word;
  }

  // the least key whose weight is p or more (the largest logit's at least)
  __device__ unsigned least_key(double p) const {
    unsigned lo = 0, hi = key_of(top);
    if (p > 1.0) return hi;
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2;
      if (weight(of_key(mid)) >= p) hi = mid; else lo = mid + 1;
    }
    return hi;
  }
};

template <typename T>
__global__ __launch_bounds__(THREADS) void sample_rows(const typename T::Storage* __restrict__ logits, SampleArgs a) {
  __shared__ Shared sh;
  const int64_t n = blockIdx.x;
  const int vocab = (int)a.vocab;
  const float t = a.temperature != nullptr ? a.temperature[n] : 1.f;
  Row<T> row = {logits + n * a.row_stride, vocab, a.bits, 0.f, 0.f, 0.0, sh};
  unsigned best = 0;
  for (int i = threadIdx.x; i < vocab; i += THREADS) best = max(best, key_of(row.at(i)));
  for (int o = 32; o > 0; o >>= 1) best = max(best, (unsigned)__shfl_xor((int)best, o));
  if ((threadIdx.x & 63) == 0) sh.counts[threadIdx.x >> 6] = best;
  __syncthreads();
  for (int w = 0; w < WAVES; w++) best = max(best, sh.counts[w]);
  __syncthreads();
  if (best <= NOTHING) {  // no number above minus infinity
    if (threadIdx.x == 0) {
      a.tokens[n] = -1;
      if (a.logprobs != nullptr) a.logprobs[n] = -__builtin_inff();
    }
    return;
  }
  if (!(t > 0.f)) {
    const int i = row.index_of(best, 1);
    if (threadIdx.x == 0) {
      a.tokens[n] = i;
      if (a.logprobs != nullptr) a.logprobs[n] = 0.f;
    }
    return;
  }
  row.top = of_key(best);
  row.inv = 1.f / t;
  row.inv64 = 1.0 / (double)t;
  row.clear(sh.mass0, sh.count0);
  uint64_t total = 0;
  for (int i = threadIdx.x; i < vocab; i += THREADS) {
    const float v = of_key(key_of(row.at(i)));
    const uint64_t w = row.whole(v);
    const int b = row.bin(v);
    total += w;
    atomicAdd(&sh.count0[b], 1u);
    atomicAdd((unsigned long long*)&sh.mass0[b], (unsigned long long)w);
  }
  total = row.sum(total);
  Border end = {0u, 0xffffffffu};
  const int k = a.top_k != nullptr ? a.top_k[n] : 0;
  if (k > 0 && k < vocab) {
    end = row.find([=](uint64_t, unsigned c) { return c >= (unsigned)k; });
    total = row.mass_of(end);
  }
  const float p = a.top_p != nullptr ? a.top_p[n] : 1.f;
  if (p < 1.f) {
    // the last one kept is the first with which the mass reaches p of the whole; the first element always is one
    const double want = fmax((double)p, 0.0) * (double)total;
    const uint64_t least = (uint64_t)ceil(want) > 1 ? (uint64_t)ceil(want) : 1;
    const Border e = row.find([=](uint64_t m, unsigned) { return m >= least; });
    if (shorter(e, end)) {
      end = e;
      total = row.mass_of(end);
    }
  }
  const float q = a.min_p != nullptr ? a.min_p[n] : 0.f;
  if (q > 0.f) {
    const Border e = {row.least_key((double)q), q > 1.f ? 1u : 0xffffffffu};  // past 1: the first alone
    if (shorter(e, end)) {
      end = e;
      total = q > 1.f ? row.mass_of(end) : row.mass_of(Border{end.key - 1, 0u});  // those of its key too
    }
  }
  const float u = a.uniforms[n];
  const double share = u > 0.f ? (double)u * (double)total : u == u ? 0.0 : (double)total;
  const uint64_t before = share < (double)total ? min((uint64_t)share, total - 1) : total - 1;
  const Border drawn = row.find([=](uint64_t m, unsigned) { return m > before; });
  const int i = row.index_of(drawn.key, drawn.taken);
  if (threadIdx.x == 0) {
    a.tokens[n] = i;
    if (a.logprobs != nullptr) a.logprobs[n] = (float)log(ldexp(row.weight(of_key(drawn.key)), a.bits) / (double)total);
  }
}

template <typename T>
int sample_of(const void* logits, const SampleArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((sample_rows<T>), dim3((unsigned)a.rows), dim3(THREADS), 0, stream, (const typename T::Storage*)logits, a);
  return check_hip(hipGetLastError(), "launching sampling");
}

}  // namespace
}  // namespace limn

using namespace limn;

extern "C" int64_t limn_hip_sample_workspace(int dtype, int64_t rows, int64_t vocab) { return 0; }

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
  if (rows > 0x7fffffff || vocab > (1 << 24)) return fail(LIMN_HIP_EUNSUPPORTED, "sample: sizes out of range");
  int log2v = 0;
  while (((int64_t)1 << log2v) < vocab) log2v++;
  const SampleArgs a = {(const float*)uniforms, (const float*)temperature, (const int*)top_k, (const float*)top_p, (const float*)min_p, (int*)tokens,
                        (float*)logprobs, rows, vocab, row_stride, 62 - log2v < 52 ? 62 - log2v : 52};
  const hipStream_t s = (hipStream_t)stream;
  return dtype == LIMN_HIP_FLOAT32 ? sample_of<F32>(logits, a, s) : dtype == LIMN_HIP_FLOAT16 ? sample_of<F16>(logits, a, s) : sample_of<BF16>(logits, a, s);
}
