// Log probabilities of given tokens, entropy and top alternatives of rows of fp32 logits.
//
//   d_j = z_j - max z      S = sum_j exp d_j      log p_t = d_t - ln S      H = ln S - (sum_j d_j exp d_j) / S
//
// One CTA of 1024 threads per row, which reads the row once for the maximum, once for the sums and once per alternative.
#include "common.cuh"
#include "logprob.cuh"

using namespace b2;

namespace {

constexpr int kThreads = 1024;

struct RowsParams {
  const float* z;      // [m][ld]
  long long ld;
  int n, top;
  const int* tokens;   // [m]
  float *logprob, *entropy;
  int* top_ids;        // [m][top]
  float* top_logprobs;
};

__global__ void __launch_bounds__(kThreads) logprob_rows_kernel(const RowsParams p) {
  __shared__ float red_f[3][32];
  __shared__ unsigned long long red_k[32];
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* z = p.z + row * p.ld;
  // the largest logit, as a key: numbers above NaN, ties to the lower id
  const auto largest_below = [&](unsigned long long bound) {
    unsigned long long best = 0;
    for (int j = threadIdx.x; j < p.n; j += kThreads) {
      const unsigned long long k = logit_key(z[j], j);
      if (k < bound && k > best) best = k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) red_k[warp] = best;
    __syncthreads();
    best = red_k[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    return best;
  };
  const unsigned long long first = largest_below(~0ull);
  const float zmax = key_id(first) < (unsigned)p.n ? z[key_id(first)] : -INFINITY;
  LogStat s{zmax, 0.f, 0.f};
  for (int j = threadIdx.x; j < p.n; j += kThreads)
    if (j != (int)key_id(first)) add_term(s, z[j]);
  s.s = warp_sum(s.s);
  s.t = warp_sum(s.t);
  if (lane == 0) {
    red_f[0][warp] = s.s;
    red_f[1][warp] = s.t;
  }
  __syncthreads();
  s.s = warp_sum(red_f[0][lane]);
  s.t = warp_sum(red_f[1][lane]);
  const LogNorm norm = log_norm(s);
  if (threadIdx.x == 0) {
    const int t = p.tokens[row];
    p.logprob[row] = t >= 0 && t < p.n ? log_prob(norm, z[t]) : NAN;
    p.entropy[row] = norm.entropy;
  }
  unsigned long long key = first;
  for (int i = 0; i < p.top; ++i) {
    if (i) key = largest_below(key);
    if (threadIdx.x == 0) {
      const bool there = i < p.n;
      p.top_ids[(long long)row * p.top + i] = there ? (int)key_id(key) : -1;
      p.top_logprobs[(long long)row * p.top + i] = there ? log_prob(norm, z[key_id(key)]) : -INFINITY;
    }
  }
}

}  // namespace

// z: [m] rows of n logits, ld elements apart.  top: alternatives per row, at most kMaxTop.
extern "C" int b2_logprob_rows(const float* z, long long ld, int m, int n, const int* tokens, int top, float* logprob, float* entropy,
                               int* top_ids, float* top_logprobs, void* stream) {
  if (m < 1 || n < 1 || ld < n || top < 0 || top > kMaxTop) return -1;
  const RowsParams p{z, ld, n, top, tokens, logprob, entropy, top_ids, top_logprobs};
  logprob_rows_kernel<<<m, kThreads, 0, (cudaStream_t)stream>>>(p);
  return (int)cudaGetLastError();
}
extern "C" int b2_logprob_max_top() { return kMaxTop; }

B2_DEFINE_STATUS(logprob)
