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
  float cap_in, cap_out; // 2 log2(e) scale / cap and cap log2(e); cap_out = 0: no cap
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
  r.cap_in = a.softcap > 0.f ? 2.f * ATT_LOG2E * a.scale / a.softcap : 0.f;
  r.cap_out = a.softcap * ATT_LOG2E;
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

// log2 of a row's normalizer; infinite for a row that sees nothing, so that its probabilities are 0
__device__ __forceinline__ float att_l2(float lse) { return lse == -__builtin_inff() ? __builtin_inff() : lse * ATT_LOG2E; }

}  // namespace
}  // namespace limn
