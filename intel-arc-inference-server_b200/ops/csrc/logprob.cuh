// What the kernels of log probabilities share: a row's maximum and sums, the order of its logits, its results.
#pragma once
#include "common.cuh"

namespace b2 {

constexpr int kMaxTop = 32;      // alternatives of a row

// Of a set of logits z: m = max z, s = sum exp(z - m) without one term of m itself, t = sum (z - m) exp(z - m).  S = 1 + s: kept apart,
// the logarithm of a sum near one keeps its digits (a token of probability 1 - 1e-8 has a log probability of -1e-8, where 1 + 1e-8 in
// fp32 is 1).  An empty set, or one of nothing but -inf, has m = -inf and s = t = 0; a NaN or a +inf among the logits makes s a NaN.
struct LogStat {
  float m, s, t;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// z - m, bounded from below: exp(-200) is 0 in fp32, and 0 times a bounded number is 0 where 0 times -inf is not.  m of a set without
// a finite number counts as the lowest one, so that -inf minus it is -inf.
__device__ __forceinline__ float below(float z, float m) { return max_nan(z - fmaxf(m, -3.402823466e38f), -200.f); }

// N more logits, the largest of them `largest`.
template <int N>
__device__ __forceinline__ void add_terms(LogStat& s, const float (&v)[N], float largest) {
  const bool record = largest > s.m;
  if (record) {      // the old maximum becomes a term like others
    if (s.m > -INFINITY) {
      const float d = below(s.m, largest), f = ex2(d * kLog2e), n = 1.f + s.s;
      s.t = f * fmaf(d, n, s.t);
      s.s = n * f;
    }
    s.m = largest;
  }
  const float m = fmaxf(s.m, -3.402823466e38f);
  float less = 0.f, equal = record ? -1.f : 0.f;      // of the maximum's own terms one is not counted
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = max_nan(v[i] - m, -200.f), e = ex2(d * kLog2e), one = d == 0.f ? 1.f : 0.f;
    less += e - one;
    equal += one;
    s.t = fmaf(d, e, s.t);
  }
  s.s += less + equal;
}

// a and b together.
__device__ __forceinline__ LogStat join(const LogStat& a, const LogStat& b) {
  const bool first = !(a.m < b.m);
  const LogStat &hi = first ? a : b, &lo = first ? b : a;
  if (lo.m == -INFINITY) return LogStat{hi.m, hi.s + lo.s, hi.t};      // nothing there (its s is 0 or a NaN)
  const float d = below(lo.m, hi.m), f = ex2(d * kLog2e), n = 1.f + lo.s;
  return LogStat{hi.m, fmaf(n, f, hi.s), hi.t + f * fmaf(d, n, lo.t)};
}

struct LogNorm {
  float m, lse, entropy;      // log p = (z - m) - lse
};
__device__ __forceinline__ LogNorm log_norm(const LogStat& s) {
  LogNorm n;
  n.m = s.m;
  n.lse = s.m < INFINITY ? log1pf(s.s) : NAN;
  n.entropy = n.lse - s.t / (1.f + s.s);
  return n;
}
__device__ __forceinline__ float log_prob(const LogNorm& n, float z) {
  if (n.m == -INFINITY) return n.lse == n.lse ? z : NAN;      // no finite logit: every probability is 0
  return (z - n.m) - n.lse;
}

// Larger logits have larger keys, of equal ones the lower id; NaN comes below -inf, and both zeros are one value.  No key is 0.
__device__ __forceinline__ uint32_t logit_order(float z) {
  const uint32_t u = __float_as_uint(z + 0.f);
  return z != z ? 1u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long logit_key(float z, int id) { return ((unsigned long long)logit_order(z) << 32) | (uint32_t)~id; }
__device__ __forceinline__ uint32_t key_id(unsigned long long key) { return ~(uint32_t)key; }

}  // namespace b2
