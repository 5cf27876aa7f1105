// The C ABI of the head's cross entropy (include/limn_hip.h): argument checks.

#include "xent.h"

namespace limn {
namespace {

int check_xent(const char* name, const XentArgs& a) {
  if (a.dtype != LIMN_HIP_FLOAT32 && a.dtype != LIMN_HIP_FLOAT16 && a.dtype != LIMN_HIP_BFLOAT16)
    return fail(LIMN_HIP_EUNSUPPORTED, "%s: takes float32, float16 or bfloat16, not dtype code %d", name, a.dtype);
  if (a.rows < 1 || a.width < 1 || a.vocab < 1)
    return fail(LIMN_HIP_EINVAL, "%s: sizes must be positive (rows %lld, width %lld, vocab %lld)", name, (long long)a.rows, (long long)a.width,
                (long long)a.vocab);
  if (a.vocab > 0x7fffffff || a.rows > ((int64_t)1 << 40) / a.width || a.vocab > ((int64_t)1 << 40) / a.width || !xent_sizes_ok(a))
    return fail(LIMN_HIP_EUNSUPPORTED, "%s: sizes out of range (operands reach past 2 GiB)", name);
  return LIMN_HIP_OK;
}

int check_call(const char* name, const XentArgs& a, bool backward) {
  int rc = check_xent(name, a);
  if (rc != LIMN_HIP_OK) return rc;
  if (a.x == nullptr || a.w == nullptr || a.targets == nullptr || a.o0 == nullptr || a.o1 == nullptr) return fail(LIMN_HIP_EINVAL, "%s: null buffer", name);
  if (backward && (a.lse_in == nullptr || a.g == nullptr)) return fail(LIMN_HIP_EINVAL, "%s: null buffer", name);
  const uintptr_t size = a.dtype == LIMN_HIP_FLOAT32 ? 4 : 2, outs = (uintptr_t)a.o0 | (uintptr_t)a.o1;
  if (((uintptr_t)a.x | (uintptr_t)a.w) % size != 0 || outs % (backward ? size : 4) != 0 || ((uintptr_t)a.targets | (uintptr_t)a.lse_in | (uintptr_t)a.g) % 4 != 0)
    return fail(LIMN_HIP_EINVAL, "%s: buffers must be aligned to their element size", name);
  const int64_t need = xent_workspace(a, backward);
  if (a.workspace == nullptr || a.workspace_bytes < need || (uintptr_t)a.workspace % 16 != 0)
    return fail(LIMN_HIP_EINVAL, "%s: needs a workspace of %lld bytes, 16-byte aligned", name, (long long)need);
  return LIMN_HIP_OK;
}

}  // namespace
}  // namespace limn

using namespace limn;

extern "C" {

int64_t limn_hip_xent_workspace(int dtype, int64_t rows, int64_t width, int64_t vocab, int backward) {
  XentArgs a = {};
  a.dtype = dtype, a.rows = rows, a.width = width, a.vocab = vocab;
  return check_xent("xent_workspace", a) == LIMN_HIP_OK ? xent_workspace(a, backward != 0) : 0;
}

int limn_hip_xent_fwd(const void* x, const void* w, const void* targets, void* loss, void* lse, int dtype, int64_t rows, int64_t width,
                      int64_t vocab, void* workspace, int64_t workspace_bytes, void* stream) {
  const XentArgs a = {x, w, (const int*)targets, nullptr, nullptr, loss, lse, dtype, rows, width, vocab, workspace, workspace_bytes, (hipStream_t)stream};
  const int rc = check_call("xent_fwd", a, false);
  return rc != LIMN_HIP_OK ? rc : launch_xent_fwd(a);
}

int limn_hip_xent_bwd(const void* x, const void* w, const void* targets, const void* lse, const void* g, void* dx, void* dw, int dtype,
                      int64_t rows, int64_t width, int64_t vocab, void* workspace, int64_t workspace_bytes, void* stream) {
  const XentArgs a = {x, w, (const int*)targets, (const float*)lse, (const float*)g, dx, dw, dtype, rows, width, vocab, workspace, workspace_bytes,
                      (hipStream_t)stream};
  const int rc = check_call("xent_bwd", a, true);
  return rc != LIMN_HIP_OK ? rc : launch_xent_bwd(a);
}

}  // extern "C"
