// The C ABI of attention over a paged cache: argument checks, choice of kernels; the write of the new tokens' keys and
// values into their pages; and the kernel that serves every type, head dim and alignment.

#include "paged_fast.h"
#include "paged_reads.h"

#include <math.h>

namespace limn {
namespace {

// A workgroup a token: its key and value rows to their places, and zeros to out where it belongs to no sequence. Bytes in
// and out, each once.
template <typename S>
__global__ __launch_bounds__(256) void paged_write(PagedView v, const S* __restrict__ k, const S* __restrict__ val, S* __restrict__ key_pages,
                                                   S* __restrict__ value_pages, S* __restrict__ out) {
  const int row = blockIdx.x, s = sequence_of(v, row);
  if (s < 0) {
    for (int i = threadIdx.x; i < v.heads * v.hd; i += 256) out[(int64_t)row * v.heads * v.hd + i] = S(0);
    return;
  }
  if (k == nullptr) return;
  const Sequence q = sequence_at(v, s);
  const int p = q.off + row - q.row0;
  if (p < 0) return;
  const int64_t place = key_place(v, s, 0, p);
  if (place < 0) return;
  const int64_t head = (int64_t)v.div.page * v.hd;
  for (int i = threadIdx.x; i < v.kv_heads * v.hd; i += 256) {
    const int h = i / v.hd, d = i - h * v.hd;
    key_pages[place + h * head + d] = k[row * v.k_row + i];
    value_pages[place + h * head + d] = val[row * v.v_row + i];
  }
}

// A wave a token and head, for every type, head dim and alignment: 64 keys at a time, a key a lane for the scores, then
// a dim a lane (4 apart by 64) for the sum of values, with the running maximum and sum of a softmax. What it costs is
// latency: a lane's loads of its key's row one after another.
template <typename T>
__global__ __launch_bounds__(256) void paged_rows(PagedView v, const typename T::Storage* __restrict__ q, const typename T::Storage* __restrict__ key_pages,
                                                  const typename T::Storage* __restrict__ value_pages, typename T::Storage* __restrict__ out) {
  __shared__ float rows[4][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t id = blockIdx.x * (int64_t)4 + wave;
  if (id >= (int64_t)v.tokens * v.heads) return;  // whole waves, and there is no barrier
  const int row = (int)(id / v.heads), head = (int)(id - (int64_t)row * v.heads), kvh = head / v.group;
  const int s = sequence_of(v, row);
  if (s < 0) return;
  const Sequence seq = sequence_at(v, s);
  const int p = seq.off + row - seq.row0, keys = min(p + 1, seq.len);
  float* mine = rows[wave];
  for (int d = lane; d < v.hd; d += 64) mine[d] = T::load(q, row * v.q_row + (int64_t)head * v.hd + d);
  __builtin_amdgcn_wave_barrier();
  float m = -__builtin_inff(), l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  const float slope = v.slopes != nullptr ? v.slopes[head] : 0.f;
  for (int k0 = 0; k0 < keys; k0 += 64) {
    const int j = k0 + lane;
    const int64_t place = j < keys ? key_place(v, s, kvh, j) : -1;
    float x = 0.f;
    if (place >= 0)
      for (int d = 0; d < v.hd; d++) x = fmaf(mine[d], T::load(key_pages, place + d), x);
    x *= v.scale;
    if (v.softcap > 0.f) x = v.softcap * tanhf(x / v.softcap);
    x = place >= 0 ? x - slope * (float)(p - j) : -__builtin_inff();
    float top = x;
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float up = fmaxf(m, top), base = up == -__builtin_inff() ? 0.f : up;
    const float old = m == -__builtin_inff() ? 1.f : expf(m - base);
    // (a score of NaN is no maximum, and its weight is NaN, as the sums then are)
    const float w = place >= 0 ? expf(x - base) : 0.f;
    float sum = w;
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    l = l * old + sum;
    m = up;
#pragma unroll
    for (int c = 0; c < 4; c++) acc[c] *= old;
    const uint64_t live = __ballot(place >= 0);
    for (int i = 0; i < 64; i++) {
      if (!((live >> i) & 1)) continue;
      const float wi = __shfl(w, i);
      const int64_t at = ((int64_t)__shfl((int)(place >> 32), i) << 32) | (unsigned)__shfl((int)place, i);
#pragma unroll
      for (int c = 0; c < 4; c++)
        if (c * 64 + lane < v.hd) {
          const float x = T::load(value_pages, at + c * 64 + lane);
          acc[c] = x - x == 0.f ? fmaf(wi, x, acc[c]) : acc[c] + x;  // (an infinity stays one under a weight that has come to 0)
        }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < 4; c++)
    if (c * 64 + lane < v.hd) T::store(out, ((int64_t)row * v.heads + head) * v.hd + c * 64 + lane, acc[c] * inv);
}

// a wave a token and head, in fours
int64_t row_blocks(const PagedArgs& a) { return (a.tokens * a.heads + 3) / 4; }

template <typename T>
int rows_of(const PagedArgs& a) {
  typedef typename T::Storage S;
  hipLaunchKernelGGL((paged_rows<T>), dim3((unsigned)row_blocks(a)), dim3(256), 0, a.stream, paged_view(a), (const S*)a.q, (const S*)a.key_pages,
                     (const S*)a.value_pages, (S*)a.out);
  return check_hip(hipGetLastError(), "launching attention over a paged cache");
}

template <typename S>
int write_of(const PagedArgs& a) {
  hipLaunchKernelGGL((paged_write<S>), dim3((unsigned)a.tokens), dim3(256), 0, a.stream, paged_view(a), (const S*)a.k, (const S*)a.v, (S*)a.key_pages,
                     (S*)a.value_pages, (S*)a.out);
  return check_hip(hipGetLastError(), "launching the write of a paged cache");
}

// ---- the tiled kernels ----

// Joins the parts of a sequence: a wave a token and head, the parts' totals brought to the largest reference point and added
// in their order. A part that saw nothing (no reference point and a sum of 0: it is NaN where a score was) counts nothing. A lane
// has a part's statistics, so that the loads do not wait for one another.
template <typename T>
__global__ __launch_bounds__(256) void paged_join(PagedFast f, PagedView v) {
  const int lane = threadIdx.x & 63;
  const int64_t id = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6), rows_all = (int64_t)v.tokens * v.heads;
  if (id >= rows_all) return;  // whole waves, and there is no barrier
  const int row = (int)(id / v.heads), s = sequence_of(v, row);
  if (s < 0) return;
  const Sequence q = sequence_at(v, s);
  const int tile = ((row - q.row0) * v.group + (int)(id - (int64_t)row * v.heads) % v.group) / f.rows;
  const int parts = (span_of(v, q, tile, f.rows, f.k != nullptr, f.keys).tiles + f.part_tiles - 1) / f.part_tiles;
  if (parts <= 1) return;
  float top = -__builtin_inff();
  for (int p = lane; p < parts; p += 64) top = fmaxf(top, f.stats[(p * rows_all + id) * 2]);
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float base = top == -__builtin_inff() ? 0.f : top;
  float total = 0.f, x[2] = {0.f, 0.f};
  for (int p0 = 0; p0 < parts; p0 += 64) {
    const int many = min(64, parts - p0);
    float w = 0.f, sum = 0.f;
    if (lane < many) {
      const float2 st = *(const float2*)&f.stats[((p0 + lane) * rows_all + id) * 2];
      w = st.x == -__builtin_inff() ? (st.y == 0.f ? 0.f : 1.f) : fast_exp2(st.x - base);
      sum = st.x == -__builtin_inff() && st.y == 0.f ? 0.f : st.y * w;
    }
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
    total += sum;
#pragma unroll 8
    for (int p = 0; p < many; p++) {
      const float wp = __shfl(w, p);
#pragma unroll
      for (int c = 0; c < 2; c++)
        if (c * 64 + lane < v.hd) {
          const float y = f.totals[((p0 + p) * rows_all + id) * v.hd + c * 64 + lane];
          x[c] += y - y == 0.f ? wp * y : y;  // (an infinity stays one under a weight that has come to 0)
        }
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
  for (int c = 0; c < 2; c++)
    if (c * 64 + lane < v.hd) T::store((typename T::Storage*)f.out + id * v.hd, c * 64 + lane, x[c] * inv);
}

int check_paged(const PagedArgs& a) {
  const char* name = "attend_paged";
  if (a.dtype != LIMN_HIP_FLOAT32 && a.dtype != LIMN_HIP_FLOAT16 && a.dtype != LIMN_HIP_BFLOAT16)
    return fail(LIMN_HIP_EUNSUPPORTED, "%s: takes float32, float16 or bfloat16, not dtype code %d", name, a.dtype);
  if (a.tokens < 1 || a.sequences < 1 || a.heads < 1 || a.kv_heads < 1 || a.hd < 1 || a.pages < 1 || a.page < 1 || a.table_pages < 1)
    return fail(LIMN_HIP_EINVAL, "%s: sizes must be positive (tokens %lld, sequences %lld, heads %lld, kv_heads %lld, hd %lld, pages %lld, page %lld, table_pages %lld)", name,
                (long long)a.tokens, (long long)a.sequences, (long long)a.heads, (long long)a.kv_heads, (long long)a.hd, (long long)a.pages, (long long)a.page,
                (long long)a.table_pages);
  if (a.heads % a.kv_heads != 0)
    return fail(LIMN_HIP_EINVAL, "%s: %lld query heads do not share %lld key heads evenly", name, (long long)a.heads, (long long)a.kv_heads);
  if (a.q_row < a.heads * a.hd || (a.k != nullptr && (a.k_row < a.kv_heads * a.hd || a.v_row < a.kv_heads * a.hd)))
    return fail(LIMN_HIP_EINVAL, "%s: rows of %lld, %lld and %lld elements overlap", name, (long long)a.q_row, (long long)a.k_row, (long long)a.v_row);
  // the kernels' constants are floats: a scale or a cap past this, or a cap below its inverse, would be an infinity or a 0 there
  const double most = 0x1p120;
  if (!(fabs(a.scale) <= most)) return fail(LIMN_HIP_EINVAL, "%s: scale must be finite, between -2^120 and 2^120", name);
  if (a.softcap != 0 && !(a.softcap >= 1 / most && a.softcap <= most))
    return fail(LIMN_HIP_EINVAL, "%s: softcap must be positive, between 2^-120 and 2^120, or 0 for none", name);
  if (a.hd > 256) return fail(LIMN_HIP_EUNSUPPORTED, "%s: no kernel for head dim %lld (at most 256)", name, (long long)a.hd);
  // positions, rows, pages and workgroups are 32-bit in the kernels; element offsets are 64-bit
  const int64_t size = (int64_t)1 << 30;
  if (a.heads > 65536 || a.sequences > (1 << 20) || a.tokens > size / a.heads || a.table_pages > size || a.page > size / a.table_pages || a.pages > size ||
      a.sequences > size / a.heads)
    return fail(LIMN_HIP_EUNSUPPORTED, "%s: sizes out of range", name);
  return LIMN_HIP_OK;
}

int check_buffers(const PagedArgs& a) {
  const char* name = "attend_paged";
  if (a.q == nullptr || a.key_pages == nullptr || a.value_pages == nullptr || a.starts == nullptr || a.lengths == nullptr || a.table == nullptr || a.out == nullptr)
    return fail(LIMN_HIP_EINVAL, "%s: null buffer", name);
  if ((a.k == nullptr) != (a.v == nullptr)) return fail(LIMN_HIP_EINVAL, "%s: new keys and new values go together", name);
  const uintptr_t size = a.dtype == LIMN_HIP_FLOAT32 ? 4 : 2;
  const uintptr_t typed = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.key_pages | (uintptr_t)a.value_pages | (uintptr_t)a.out;
  const uintptr_t words = (uintptr_t)a.starts | (uintptr_t)a.lengths | (uintptr_t)a.table | (uintptr_t)a.slopes;
  if (typed % size != 0 || words % 4 != 0) return fail(LIMN_HIP_EINVAL, "%s: buffers must be aligned to their element size", name);
  if (a.workspace_bytes < 0) return fail(LIMN_HIP_EINVAL, "%s: negative workspace size", name);
  return LIMN_HIP_OK;
}

template <typename T>
int join_of(const PagedArgs& a, const PagedFast& f) {
  hipLaunchKernelGGL((paged_join<T>), dim3((unsigned)row_blocks(a)), dim3(256), 0, a.stream, f, paged_view(a));
  return check_hip(hipGetLastError(), "joining the parts of attention over a paged cache");
}

// Sizes that the tiled kernels serve: rows of whole 16-byte chunks; places counted in 32 bits.
bool fast_sizes(const PagedArgs& a) {
  return paged_dim(a.hd, a.dtype == LIMN_HIP_FLOAT32 ? 4 : 2) && a.pages < (int64_t)0xffffffff / a.kv_heads / a.page;
}
// A call of such sizes goes to them where every buffer and row is 16-byte aligned, and its constants stay normal numbers.
bool fast_call(const PagedArgs& a) {
  const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.key_pages | (uintptr_t)a.value_pages | (uintptr_t)a.out;
  const int64_t per = a.dtype == LIMN_HIP_FLOAT32 ? 4 : 8;
  return fast_sizes(a) && at % 16 == 0 && a.q_row % per == 0 && (a.k == nullptr || (a.k_row % per == 0 && a.v_row % per == 0 && a.k_row < (1 << 29) && a.v_row < (1 << 29)));
}

// How a call is run: by paged_tiles (half widths) or paged_token, and in how many parts.
struct Plan {
  bool tiled, lone;
  int rows, parts, part_tiles;
};

// parts of `tiles` key tiles that bring `units` workgroups to `fill`, each at least 8 tiles
void cut(Plan& p, int64_t tiles, int64_t units, int64_t fill) {
  int64_t n = fill / (units > 1 ? units : 1);
  if (n > tiles / 8) n = tiles / 8;
  if (n < 1) n = 1;
  p.part_tiles = (int)((tiles + n - 1) / n);
  p.parts = (int)((tiles + p.part_tiles - 1) / p.part_tiles);
}

// paged_token takes the calls that have a token a sequence or fewer, or few rows in all; paged_tiles the others, in which
// any sequence may have many (how many each has is known on the device alone). 24 single tokens beside two parts of 500:
// 58 us by paged_tiles alone, 73 with a launch of each kernel for its own sequences; 32 single tokens 180 us by paged_tiles, 156 by
// paged_token.
constexpr int FEW_ROWS = 64;

Plan plan_of(const PagedArgs& a, bool tiled) {
  Plan p;
  const int64_t places = a.table_pages * a.page, all = a.tokens * a.group(), each = (a.tokens + a.sequences - 1) / a.sequences * a.group();
  p.tiled = tiled && a.dtype != LIMN_HIP_FLOAT32 && a.tokens > a.sequences && all > FEW_ROWS;
  p.lone = false;
  // In parts for 256, 512, 768, 1024 and 1536 workgroups, us: 24 single tokens beside two parts of 500 96, 72, 52, 57 and 56; 8 beside one of
  // 1000, one key head, 16000 positions 171, 93, 78, 95, 86; a part alone of 256 tokens against 8192 positions, 8 key heads 96, 67, 81, 79,
  // 76; of 2048, 2 key heads 244, 123, 129, 117, 121; of 128 against 32768, 8 key heads of 64 dims 59, 44, 44, 44, 44; of 512 against 16384,
  // one key head 56, 55, 55, 55, 54. Two workgroups share a CU, so 512 is one round of equal workgroups, which a part alone has; in a
  // mixed batch most slots are short or empty, and 768 even them out. What a batch holds is known on the device alone.
  if (p.tiled) {
    p.rows = 128;
    cut(p, (places + 63) / 64 + 1, (a.sequences + all / 128) * a.kv_heads, 768);
    return p;
  }
  // Row tiles of 16 where one holds a sequence's packed rows, else of 32. Up to 64 key tiles go to one workgroup of many waves a
  // row tile while such workgroups leave waves free; longer caches to workgroups of 4 waves, two a CU. (32 tokens over up to 8192
  // positions, 8 key heads, in parts for 512, 768, 1024 and 2048 workgroups: 156, 172, 167 and 185 us.)
  const int64_t tiles = (places + 31) / 32 + 1;
  p.rows = each <= 16 ? 16 : 32;
  const int64_t units = a.sequences * a.kv_heads * ((each + p.rows - 1) / p.rows);
  p.lone = tiles <= 65 && units <= 256;
  cut(p, tiles, units, p.lone ? 1 : 512);
  return p;
}

constexpr int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Whether the scale fits paged_tiles: it multiplies a tile's maximum behind the products, and must be a normal number above 0.
bool tile_scale(const PagedArgs& a) { return a.scale >= 0x1p-100; }

// Enough whatever the call's scale and alignment.
int64_t workspace_of(const PagedArgs& a) {
  if (!fast_sizes(a)) return 0;
  const int64_t tiled = plan_of(a, true).parts, other = plan_of(a, false).parts, parts = tiled > other ? tiled : other, rows = a.tokens * a.heads;
  return parts > 1 ? align256(parts * rows * a.hd * 4) + align256(parts * rows * 8) : 0;
}

int launch_fast(const PagedArgs& a) {
  const Plan p = plan_of(a, tile_scale(a));
  PagedFast f = {a.q, a.k, a.v, a.key_pages, a.value_pages, a.out, nullptr, nullptr, p.parts, p.part_tiles, p.rows, p.tiled ? 64 : 32};
  if (p.parts > 1) {
    f.totals = (float*)a.workspace;
    f.stats = (float*)((char*)a.workspace + align256(p.parts * a.tokens * a.heads * a.hd * 4));
  }
  const int rc = !p.tiled        ? launch_paged_token(a, f, p.lone)
                 : a.hd <= 64 ? launch_paged_tiles_64(a, f)
                 : a.hd <= 96 ? launch_paged_tiles_96(a, f)
                              : launch_paged_tiles_128(a, f);
  if (rc != LIMN_HIP_OK || p.parts == 1) return rc;
  return a.dtype == LIMN_HIP_FLOAT32 ? join_of<F32>(a, f) : a.dtype == LIMN_HIP_FLOAT16 ? join_of<F16>(a, f) : join_of<BF16>(a, f);
}

}  // namespace
}  // namespace limn

using namespace limn;

extern "C" int64_t limn_hip_attend_paged_workspace(int dtype, int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t hd, int64_t pages,
                                                   int64_t page, int64_t table_pages) {
  const PagedArgs a = {nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, dtype, tokens, sequences, heads, kv_heads, hd, pages,
                       page, table_pages, heads * hd, 0, 0, 1.0, 0.0, nullptr, 0, nullptr};
  return check_paged(a) == LIMN_HIP_OK ? workspace_of(a) : 0;
}

extern "C" int limn_hip_attend_paged(const void* q, const void* k, const void* v, void* key_pages, void* value_pages, const void* starts, const void* lengths,
                                     const void* table, const void* slopes, void* out, int dtype, int64_t tokens, int64_t sequences, int64_t heads,
                                     int64_t kv_heads, int64_t hd, int64_t pages, int64_t page, int64_t table_pages, int64_t q_row, int64_t k_row,
                                     int64_t v_row, double scale, double softcap, void* workspace, int64_t workspace_bytes, void* stream) {
  const PagedArgs a = {q, k, v, key_pages, value_pages, (const int*)starts, (const int*)lengths, (const int*)table, (const float*)slopes, out, dtype, tokens, sequences,
                       heads, kv_heads, hd, pages, page, table_pages, q_row, k_row, v_row, scale, softcap, workspace, workspace_bytes, (hipStream_t)stream};
  int rc = check_paged(a);
  if (rc == LIMN_HIP_OK) rc = check_buffers(a);
  if (rc != LIMN_HIP_OK) return rc;
  const int64_t need = workspace_of(a);
  if (need > 0 && (workspace == nullptr || (uintptr_t)workspace % 16 != 0 || workspace_bytes < need))
    return fail(LIMN_HIP_EINVAL, "attend_paged: needs a workspace of %lld bytes, 16-byte aligned", (long long)need);
  if (fast_call(a)) return launch_fast(a);
  const int64_t blocks = row_blocks(a) > tokens ? row_blocks(a) : tokens;  // before anything is written
  if (!one_launch(blocks, 256)) return fail(LIMN_HIP_EUNSUPPORTED, "attend_paged: sizes out of range, %lld workgroups exceed one launch", (long long)blocks);
  rc = dtype == LIMN_HIP_FLOAT32 ? write_of<float>(a) : write_of<u16>(a);
  if (rc != LIMN_HIP_OK) return rc;
  return dtype == LIMN_HIP_FLOAT32 ? rows_of<F32>(a) : dtype == LIMN_HIP_FLOAT16 ? rows_of<F16>(a) : rows_of<BF16>(a);
}
