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

constexpr float kLog2e = 1.4426950408889634f;

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

__device__ __forceinline__ float order_value(uint32_t o) {      // of logit_order
  return __uint_as_float(o == 1u ? 0x7fffffffu : (o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
}

// The stats of `width` lanes (a power of two) in all of them: the maximum first, then plain sums of what each lane is to it.
template <int width>
__device__ __forceinline__ LogStat join_lanes(const LogStat& a) {
  float m = a.m;
#pragma unroll
  for (int o = width / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const bool none = a.m == -INFINITY, best = a.m == m;
  const float d = below(a.m, m), f = ex2(d * kLog2e), n = 1.f + a.s;
  LogStat r{m, none || best ? a.s : n * f, none || best ? a.t : f * fmaf(d, n, a.t)};
  float count = best && !none ? 1.f : 0.f;      // lanes with a term of the maximum beside their sums
#pragma unroll
  for (int o = width / 2; o > 0; o >>= 1) {
    r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
    r.t += __shfl_xor_sync(0xffffffffu, r.t, o);
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
  r.s += fmaxf(count - 1.f, 0.f);
  return r;
}

// The largest 32 keys of two lists, each sorted across the lanes, the largest first; so is the result.
__device__ __forceinline__ unsigned long long merge_lists(unsigned long long a, unsigned long long b, int lane) {
  unsigned long long k = max(a, __shfl_xor_sync(0xffffffffu, b, 31));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
    k = (lane & o) ? min(k, other) : max(k, other);
  }
  return k;
}

// One more key for a sorted list.
__device__ __forceinline__ void insert(unsigned long long& list, unsigned long long key, int lane) {
  const int at = __popc(__ballot_sync(0xffffffffu, list > key));
  const unsigned long long before = __shfl_up_sync(0xffffffffu, list, 1);
  list = lane < at ? list : lane == at ? key : before;
}

// The lanes' numbers, none of them NaN, the largest first.
__device__ __forceinline__ float sort_lanes(float x, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, x, o);
      const bool low = (lane & o) == 0, falling = (lane & size) == 0;
      x = low == falling ? fmaxf(x, other) : fminf(x, other);
    }
  return x;
}
// The largest 32 of two lists of numbers, as merge_lists.
__device__ __forceinline__ float merge_floats(float a, float b, int lane) {
  float x = fmaxf(a, __shfl_xor_sync(0xffffffffu, b, 31));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, x, o);
    x = (lane & o) ? fminf(x, other) : fmaxf(x, other);
  }
  return x;
}

// A list with fewer than `top` logits above -inf: banned ids follow, the lowest first, then those without a number.
__device__ __forceinline__ unsigned long long fill_list(unsigned long long list, const float* z, int n, int top, int lane) {
  int have = __popc(__ballot_sync(0xffffffffu, list != 0));
  constexpr int kAhead = 8;
  for (int kind = 0; kind < 2 && have < top; ++kind) {
    for (int j0 = 0; j0 < n && have < top; j0 += 32 * kAhead) {
      float x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) x[i] = j0 + 32 * i + lane < n ? z[j0 + 32 * i + lane] : 0.f;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int first = j0 + 32 * i;
        const uint32_t mask = __ballot_sync(0xffffffffu, first + lane < n && (kind == 0 ? x[i] == -INFINITY : x[i] != x[i]));
        const int nth = lane - have;      // this lane's place is the nth of them
        if (nth >= 0 && nth < __popc(mask)) list = logit_key(kind == 0 ? -INFINITY : __int_as_float(0x7fffffff), first + __fns(mask, 0, nth + 1));
        have += __popc(mask);
      }
    }
  }
  return list;
}

// A logit per lane into a sorted list of which the first `top` count; last: the top-th key.
__device__ __forceinline__ void offer(unsigned long long& list, unsigned long long& last, unsigned long long key, int top, int lane) {
  uint32_t more = __ballot_sync(0xffffffffu, key > last);
  while (more) {
    insert(list, __shfl_sync(0xffffffffu, key, __ffs(more) - 1), lane);
    last = __shfl_sync(0xffffffffu, list, top - 1);
    more = __ballot_sync(0xffffffffu, key > last) & (more & (more - 1));
  }
}

}  // namespace b2
