// Internal launch interface of the head's cross entropy (xent_tiles.hip).
#pragma once

#include "matmul.h"

namespace limn {

// loss[n] = logsumexp_v(x[n] . w[v]) - x[n] . w[target[n]], 0 for a target outside [0, vocab); its gradients for
// cotangents g[n]: dx = dz w and dw = dz^T x with dz[n, v] = g[n] (exp(x[n] . w[v] - lse[n]) - [v = target[n]]).
struct XentArgs {
  const void* x;        // (rows, width)
  const void* w;        // (vocab, width)
  const int* targets;   // (rows)
  const float* lse_in;  // backward
  const float* g;       // backward
  void* o0;             // loss / dx
  void* o1;             // lse / dw
  int dtype;
  int64_t rows, width, vocab;
  void* workspace;
  int64_t workspace_bytes;
  hipStream_t stream;
};

constexpr int64_t xent_align(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Parts of a workspace, taken one after another.
struct XentSpace {
  char* at;
  explicit XentSpace(void* p) : at((char*)p) {}
  void* take(int64_t bytes) {
    void* p = at;
    at += xent_align(bytes);
    return p;
  }
};

bool xent_sizes_ok(const XentArgs& a);  // whether the sizes fit the kernels' 32-bit offsets
int64_t xent_workspace(const XentArgs& a, bool backward);
int launch_xent_fwd(const XentArgs& a);
int launch_xent_bwd(const XentArgs& a);

}  // namespace limn
