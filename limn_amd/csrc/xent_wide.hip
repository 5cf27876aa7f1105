// The head's cross entropy in float32 arithmetic, for every type, width and alignment.
//
// The vocabulary goes by in pieces: a piece's logits are one contraction (float32 on matrix cores,
// matmul_f32.hip) into a buffer of at most PIECE_BYTES, small enough that what reads it next finds most of
// it in the 256 MiB last-level cache; a row's running maximum and sum take the piece in, and the backward
// turns it in place into dz, which two contractions then multiply by the piece's weights (added to dx) and
// by the rows (the piece's dw). Half widths are widened to float32 copies first, a piece of the weight at a
// time. Bound by the float matrix rate; the passes over a piece move 8 bytes (forward) and 8 (backward)
// per logit beside 2 (6) width operations.

#include "xent.h"

namespace limn {
namespace {

constexpr int64_t PIECE_BYTES = (int64_t)128 << 20;

bool half(const XentArgs& a) { return a.dtype != LIMN_HIP_FLOAT32; }

int64_t piece_of(const XentArgs& a) {
  int64_t v = PIECE_BYTES / 4 / a.rows;
  v = v < 1024 ? 1024 : v / 1024 * 1024;
  return v < a.vocab ? v : a.vocab;
}

template <typename T>
__global__ __launch_bounds__(256) void widen(const typename T::Storage* __restrict__ src, float* __restrict__ dst, int64_t n) {
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) dst[i] = T::load(src, i);
}

template <typename T>
__global__ __launch_bounds__(256) void narrow(const float* __restrict__ src, typename T::Storage* __restrict__ dst, int64_t n) {
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) T::store(dst, i, src[i]);
}

// The rows with zeros in place of those without a target, which so add nothing to dw whatever they hold.
template <typename T>
__global__ __launch_bounds__(256) void live_rows(const typename T::Storage* __restrict__ x, const int* __restrict__ targets,
                                                 float* __restrict__ dst, int64_t n, int64_t width, int64_t vocab) {
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int t = targets[i / width];
    dst[i] = t >= 0 && t < vocab ? T::load(x, i) : 0.f;
  }
}

unsigned spread(int64_t n) {
  const int64_t blocks = (n + 255) / 256;
  return (unsigned)(blocks < 1 ? 1 : blocks < 8192 ? blocks : 8192);
}

int widen_to(const XentArgs& a, const void* src, float* dst, int64_t n) {
  if (a.dtype == LIMN_HIP_FLOAT16)
    hipLaunchKernelGGL((widen<F16>), dim3(spread(n)), dim3(256), 0, a.stream, (const u16*)src, dst, n);
  else
    hipLaunchKernelGGL((widen<BF16>), dim3(spread(n)), dim3(256), 0, a.stream, (const u16*)src, dst, n);
  return check_hip(hipGetLastError(), "widening an operand");
}

int narrow_to(const XentArgs& a, const float* src, void* dst, int64_t n) {
  if (a.dtype == LIMN_HIP_FLOAT16)
    hipLaunchKernelGGL((narrow<F16>), dim3(spread(n)), dim3(256), 0, a.stream, src, (u16*)dst, n);
  else
    hipLaunchKernelGGL((narrow<BF16>), dim3(spread(n)), dim3(256), 0, a.stream, src, (u16*)dst, n);
  return check_hip(hipGetLastError(), "rounding a gradient");
}

// A workgroup takes one row of a piece into the row's state (reference point, sum, target's logit): each
// thread keeps a running maximum and sum, joined in a fixed tree.
__global__ __launch_bounds__(256) void take_piece(const float* __restrict__ z, const int* __restrict__ targets, float* __restrict__ top,
                                                  float* __restrict__ sum, float* __restrict__ picked, int64_t v0, int64_t piece,
                                                  int64_t width, int first) {
  const int64_t row = blockIdx.x;
  const float* p = z + row * width;
  float m = -__builtin_inff(), l = 0.f;
  for (int64_t i = threadIdx.x; i < piece; i += 256) {
    const float x = p[i];
    if (x > m) {
      l = l * expf(m - x) + 1.f;
      m = x;
    } else {
      l += m == -__builtin_inff() ? (x == x ? 0.f : x) : expf(x - m);
    }
  }
  __shared__ float sm[256], sl[256];
  sm[threadIdx.x] = m;
  sl[threadIdx.x] = l;
  __syncthreads();
  for (int s = 128; s > 0; s >>= 1) {
    if (threadIdx.x < s) {
      const float m0 = sm[threadIdx.x], m1 = sm[threadIdx.x + s], t = fmaxf(m0, m1);
      sl[threadIdx.x] = t == -__builtin_inff() ? sl[threadIdx.x] + sl[threadIdx.x + s]
                                               : sl[threadIdx.x] * expf(m0 - t) + sl[threadIdx.x + s] * expf(m1 - t);
      sm[threadIdx.x] = t;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    m = sm[0];
    l = sl[0];
    if (!first) {
      const float m0 = top[row], t = fmaxf(m0, m);
      if (t != -__builtin_inff()) l = sum[row] * expf(m0 - t) + l * expf(m - t);
      m = t;
    }
    top[row] = m;
    sum[row] = l;
    const int64_t t = targets[row] - v0;
    if (first) picked[row] = 0.f;
    if (t >= 0 && t < piece) picked[row] = p[t];
  }
}

__global__ __launch_bounds__(256) void finish_rows(const float* __restrict__ top, const float* __restrict__ sum, const float* __restrict__ picked,
                                                   const int* __restrict__ targets, float* __restrict__ loss, float* __restrict__ lse,
                                                   int64_t rows, int64_t vocab) {
  const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
  if (i >= rows) return;
  const float l = top[i] + logf(sum[i]);
  const int t = targets[i];
  lse[i] = l;
  loss[i] = t >= 0 && t < vocab ? l - picked[i] : 0.f;
}

// a piece's logits into dz, in place
__global__ __launch_bounds__(256) void dlogits(float* __restrict__ z, const int* __restrict__ targets, const float* __restrict__ lse,
                                               const float* __restrict__ g, int64_t v0, int64_t piece, int64_t vocab) {
  const int64_t row = blockIdx.x;
  const int t = targets[row];
  const bool live = t >= 0 && t < vocab;
  const float l = lse[row], s = g[row];
  float* p = z + row * piece;
  for (int64_t i = threadIdx.x; i < piece; i += 256) p[i] = live ? s * (expf(p[i] - l) - (v0 + i == t ? 1.f : 0.f)) : 0.f;
}

MatmulShape logits_shape(const XentArgs& a, int64_t piece) {
  return {1, a.rows, piece, a.width, 0, a.width, 1, 0, 1, a.width, 0, piece, 1};
}
MatmulShape dx_shape(const XentArgs& a, int64_t piece) { return {1, a.rows, a.width, piece, 0, piece, 1, 0, a.width, 1, 0, a.width, 1}; }
MatmulShape dw_shape(const XentArgs& a, int64_t piece) { return {1, piece, a.width, a.rows, 0, 1, piece, 0, a.width, 1, 0, a.width, 1}; }

int64_t most(int64_t a, int64_t b) { return a > b ? a : b; }

// the workspace of the contractions: the last piece may be smaller, and splits otherwise than the others
int64_t product_bytes(const XentArgs& a, bool backward) {
  const int64_t piece = piece_of(a), tail = a.vocab % piece;
  int64_t need = 0;
  for (const int64_t p : {piece, tail}) {
    if (p == 0) continue;
    need = most(need, f32_workspace_bytes(logits_shape(a, p)));
    if (backward) need = most(need, most(f32_workspace_bytes(dx_shape(a, p)), f32_workspace_bytes(dw_shape(a, p))));
  }
  return need;
}

}  // namespace

bool xent_wide_ok(const XentArgs& a) {
  const int64_t piece = piece_of(a);
  return a.rows < ((int64_t)1 << 30) && a.width < ((int64_t)1 << 30) && f32_layout_ok(logits_shape(a, piece)) && f32_layout_ok(dx_shape(a, piece)) &&
         f32_layout_ok(dw_shape(a, piece));
}

int64_t xent_wide_workspace(const XentArgs& a, bool backward) {
  const int64_t piece = piece_of(a);
  int64_t need = xent_align(a.rows * piece * 4) + xent_align(product_bytes(a, backward));
  if (!backward) need += 3 * xent_align(a.rows * 4);
  if (backward || half(a)) need += xent_align(a.rows * a.width * 4);                      // the live rows (the rows, widened)
  if (half(a)) need += (1 + backward) * xent_align(piece * a.width * 4);                  // weights (and their gradients)
  if (half(a) && backward) need += xent_align(a.rows * a.width * 4);                      // dx
  return need;
}

int launch_xent_wide_fwd(const XentArgs& a) {
  const int64_t piece = piece_of(a), product = product_bytes(a, false);
  XentSpace space(a.workspace);
  float* z = (float*)space.take(a.rows * piece * 4);
  void* ws = space.take(product);
  float *top = (float*)space.take(a.rows * 4), *sum = (float*)space.take(a.rows * 4), *picked = (float*)space.take(a.rows * 4);
  const float* x = (const float*)a.x;
  float* wide = nullptr;
  int rc = LIMN_HIP_OK;
  if (half(a)) {
    float* wx = (float*)space.take(a.rows * a.width * 4);
    wide = (float*)space.take(piece * a.width * 4);
    x = wx;
    if ((rc = widen_to(a, a.x, wx, a.rows * a.width)) != LIMN_HIP_OK) return rc;
  }
  for (int64_t v0 = 0; v0 < a.vocab; v0 += piece) {
    const int64_t n = a.vocab - v0 < piece ? a.vocab - v0 : piece;
    const float* w = wide;
    if (half(a))
      rc = widen_to(a, (const u16*)a.w + v0 * a.width, wide, n * a.width);
    else
      w = (const float*)a.w + v0 * a.width;
    if (rc == LIMN_HIP_OK) rc = launch_matmul_f32(x, w, z, logits_shape(a, n), MATMUL_EPILOGUE_NONE, MatmulAddends{}, ws, product, a.stream);
    if (rc != LIMN_HIP_OK) return rc;
    hipLaunchKernelGGL(take_piece, dim3((unsigned)a.rows), dim3(256), 0, a.stream, z, a.targets, top, sum, picked, v0, n, n, (int)(v0 == 0));
    if ((rc = check_hip(hipGetLastError(), "launching the cross entropy's sums")) != LIMN_HIP_OK) return rc;
  }
  hipLaunchKernelGGL(finish_rows, dim3((unsigned)((a.rows + 255) / 256)), dim3(256), 0, a.stream, top, sum, picked, a.targets, (float*)a.o0,
                     (float*)a.o1, a.rows, a.vocab);
  return check_hip(hipGetLastError(), "launching the cross entropy's losses");
}

int launch_xent_wide_bwd(const XentArgs& a) {
  const int64_t piece = piece_of(a), product = product_bytes(a, true), rows_n = a.rows * a.width;
  XentSpace space(a.workspace);
  float* z = (float*)space.take(a.rows * piece * 4);
  void* ws = space.take(product);
  float* x = (float*)space.take(rows_n * 4);
  float *wide = nullptr, *dwide = nullptr, *dx = (float*)a.o0;
  if (half(a)) {
    wide = (float*)space.take(piece * a.width * 4);
    dwide = (float*)space.take(piece * a.width * 4);
    dx = (float*)space.take(rows_n * 4);
  }
  if (a.dtype == LIMN_HIP_FLOAT32)
    hipLaunchKernelGGL((live_rows<F32>), dim3(spread(rows_n)), dim3(256), 0, a.stream, (const float*)a.x, a.targets, x, rows_n, a.width, a.vocab);
  else if (a.dtype == LIMN_HIP_FLOAT16)
    hipLaunchKernelGGL((live_rows<F16>), dim3(spread(rows_n)), dim3(256), 0, a.stream, (const u16*)a.x, a.targets, x, rows_n, a.width, a.vocab);
  else
    hipLaunchKernelGGL((live_rows<BF16>), dim3(spread(rows_n)), dim3(256), 0, a.stream, (const u16*)a.x, a.targets, x, rows_n, a.width, a.vocab);
  int rc = check_hip(hipGetLastError(), "launching the cross entropy's rows");
  if (rc != LIMN_HIP_OK) return rc;
  for (int64_t v0 = 0; v0 < a.vocab; v0 += piece) {
    const int64_t n = a.vocab - v0 < piece ? a.vocab - v0 : piece;
    const float* w = half(a) ? wide : (const float*)a.w + v0 * a.width;
    float* dw = half(a) ? dwide : (float*)a.o1 + v0 * a.width;
    if (half(a)) rc = widen_to(a, (const u16*)a.w + v0 * a.width, wide, n * a.width);
    if (rc == LIMN_HIP_OK) rc = launch_matmul_f32(x, w, z, logits_shape(a, n), MATMUL_EPILOGUE_NONE, MatmulAddends{}, ws, product, a.stream);
    if (rc != LIMN_HIP_OK) return rc;
    hipLaunchKernelGGL(dlogits, dim3((unsigned)a.rows), dim3(256), 0, a.stream, z, a.targets, a.lse_in, a.g, v0, n, a.vocab);
    if ((rc = check_hip(hipGetLastError(), "launching the cross entropy's gradient")) != LIMN_HIP_OK) return rc;
    // later pieces add to dx: each of its elements is read and written by the one thread that owns it
    MatmulAddends add = {};
    if (v0 > 0) add = {nullptr, 0, 0, dx, 0, a.width, 1, 0};
    rc = launch_matmul_f32(z, w, dx, dx_shape(a, n), MATMUL_EPILOGUE_NONE, add, ws, product, a.stream);
    if (rc == LIMN_HIP_OK) rc = launch_matmul_f32(z, x, dw, dw_shape(a, n), MATMUL_EPILOGUE_NONE, MatmulAddends{}, ws, product, a.stream);
    if (rc == LIMN_HIP_OK && half(a)) rc = narrow_to(a, dwide, (u16*)a.o1 + v0 * a.width, n * a.width);
    if (rc != LIMN_HIP_OK) return rc;
  }
  return half(a) ? narrow_to(a, dx, a.o0, rows_n) : LIMN_HIP_OK;
}

}  // namespace limn
