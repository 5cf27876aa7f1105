// Attention with score rules: which keys a query sees and what its scores become. Shared by every
// kernel of the family.
//
//   p(i) = len - t_q + i,   s = cap tanh(scale q.k / cap) - slope |p(i) - j|
//   visible(i, j) = j < len and (not causal or j <= p(i) or j < prefix)
//                   and (no documents or (p(i) >= 0 and doc[p(i)] = doc[j] >= 0))
//
// Scores are kept in units of log2: y = s log2(e), so that a probability is one v_exp_f32.
#pragma once

#include "attend.h"

namespace limn {

struct RuleArgs {
  const float* slopes;
  const int* documents;
  const int* prefix;
  const int* lengths;
  int t_q, t_k;
  int causal;
  float scale, softcap;
};

inline RuleArgs rule_args(const AttendArgs& a) {
  return RuleArgs{a.slopes, a.documents, a.prefix, a.lengths, (int)a.t_q, (int)a.t_k, a.causal, (float)a.scale, (float)a.softcap};
}

namespace {

constexpr float ATT_LOG2E = 1.4426950408889634f, ATT_LN2 = 0.6931471805599453f;

// The rules of one sequence, and the score constants of the call.
struct Rules {
  int len, off, pre;     // live keys; position of query 0; keys below `pre` are seen whatever the order
  int t_q, t_k;
  const int* docs;       // this sequence's documents or nullptr
  bool causal;
  float c2;              // scale * log2(e)
  float cap_z, cap_in;   // |scale| / cap, and 2 log2(e) times that
  float cap_out, cap_un; // cap log2(e), 0: no cap; and its inverse
};

__device__ __forceinline__ Rules rules_of(const RuleArgs& a, int64_t b) {
  Rules r;
  int len = a.lengths ? a.lengths[b] : a.t_k;
  r.len = len < 0 ? 0 : len > a.t_k ? a.t_k : len;  // a length outside the cache never reads outside it
  r.off = r.len - a.t_q;
  r.pre = a.prefix ? a.prefix[b] : 0;
  r.t_q = a.t_q;
  r.t_k = a.t_k;
  r.docs = a.documents ? a.documents + b * a.t_k : nullptr;
  r.causal = a.causal != 0;
  r.c2 = a.scale * ATT_LOG2E;
  // (a largest number in place of an infinity: the score 0 stays 0)
  r.cap_z = a.softcap > 0.f ? fminf(fabsf(a.scale) / a.softcap, 1e38f) : 0.f;
  r.cap_in = 2.f * ATT_LOG2E * r.cap_z;
  r.cap_out = a.softcap * ATT_LOG2E;
  r.cap_un = a.softcap > 0.f ? 1.f / r.cap_out : 0.f;
  return r;
}

// A query's document: -1 where it has none (before the sequence's start, padding), which sees nothing.
__device__ __forceinline__ int query_doc(const Rules& r, int p) {
  if (r.docs == nullptr) return 0;
  if (p < 0 || p >= r.t_k) return -1;
  return r.docs[p];
}

__device__ __forceinline__ bool sees(const Rules& r, int p, int key) {
  bool ok = key < r.len;
  if (r.causal) ok &= (key <= p) | (key < r.pre);
  return ok;
}

// Products x, N of them, into capped scores in log2 units, cap_out tanh(z) with z = scale x / cap: to some 12 half steps of the
// score, however small it is beside the cap. (1 - 2 / (1 + e^2z) alone is off by half steps of the cap.) Up to |z| =
// 1/2, tanh(z) / z as a polynomial of z^2, the one of its degree with the least largest relative error, 2^-25.9; beyond,
// 1 - 2 / (1 + e^2|z|) with z's sign. A wave whose scores are all near, as they are where the cap is for outliers, takes
// neither exponential nor reciprocal.
template <int N, typename SCORES>
__device__ __forceinline__ void cap_scores(SCORES& s, const Rules& r) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < N; i++) most = fmaxf(most, fabsf(s[i]));
  auto near = [&](float x) __attribute__((always_inline)) {
    const float z = x * r.cap_z, u = z * z;
    const float p = fmaf(fmaf(fmaf(0.01724149f, u, -0.05304549f), u, 0.13325879f), u, -0.33333144f);
    return x * r.c2 * fmaf(p, u, 1.f);
  };
  if (!__any(most * r.cap_z > 0.5f)) {
#pragma unroll
    for (int i = 0; i < N; i++) s[i] = near(s[i]);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float x = s[i], w = __builtin_amdgcn_rcpf(1.f + fast_exp2(fabsf(x) * r.cap_in));
    s[i] = fabsf(x) * r.cap_z <= 0.5f ? near(x) : copysignf(fmaf(-2.f * r.cap_out, w, r.cap_out), x * r.c2);
  }
}

// What the cap takes off the gradient of a capped score y: 1 - tanh^2.
__device__ __forceinline__ float cap_slope(const Rules& r, float y) {
  const float t = y * r.cap_un;
  return fmaf(-t, t, 1.f);
}

// log2 of a row's normalizer; infinite for a row that sees nothing, so that its probabilities are 0
__device__ __forceinline__ float att_l2(float lse) { return lse == -__builtin_inff() ? __builtin_inff() : lse * ATT_LOG2E; }

}  // namespace
}  // namespace limn
