// Log probabilities of given tokens, entropy and top alternatives of rows of fp32 logits.
//
//   d_j = z_j - max z      S = sum_j exp d_j      log p_t = d_t - ln S      H = ln S - (sum_j d_j exp d_j) / S
//
// One pass over a row: its logits go through registers once, each thread with a maximum and sums of its own (LogStat).  A cluster of up
// to 16 CTAs shares a row and joins its results in the first CTA's shared memory: no workspace, no counters, the same order of every sum
// in every run.
//
// Alternatives: the top-th largest of the threads' maxima is a bound that at least `top` logits of the CTA reach, so only the logits of the
// threads whose maximum reaches it can matter: about `top` threads of a CTA, and of their logits those of the tiles (in up to eight groups)
// whose own maximum does.  Those few are read again, and what reaches the bound is put in order.  The pass itself does nothing for the
// alternatives but to keep eight maxima a thread.
// Bound by the logits' bytes with many rows (500 x 151936: 57 us with 10 alternatives, 52 without, 46 at the measured copy rate), by its own
// chain of reductions with few (1 x 151936: 7.2 and 3.9 us).  Alternatives kept in sorted lists during the pass: 108 us and 8.9.
#include "common.cuh"
#include "logprob.cuh"
#include "pair.cuh"

using namespace b2;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kVecs = 4;                              // 16-byte vectors of a thread and tile
constexpr int kTile = kThreads * kVecs;               // vectors
constexpr int kGroups = 8;                            // of a CTA's tiles
constexpr int kParts = 16;                            // CTAs that share a row, at most

struct RowsParams {
  const float* z;      // [m][ld]
  long long ld;
  int n, top, parts;
  const int* tokens;   // [m]
  float *logprob, *entropy;
  int* top_ids;        // [m][top]
  float* top_logprobs;
};

struct Shared {
  LogStat stat[kWarps], parts[kParts];
  unsigned long long list[kWarps][32], part_list[kParts][32];
  float best[kWarps][32], group[kGroups][kThreads];
  int count, chosen[kGroups * kThreads];      // group * kThreads + thread
};

__device__ __forceinline__ uint32_t map_cluster(uint32_t addr, int rank) {      // a CTA's copy of a shared-memory word
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

template <bool TOP>
__global__ void __launch_bounds__(kThreads, 4) logprob_rows_kernel(const RowsParams p) {
  __shared__ Shared sh;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (p.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // the first CTA is there: waited for below
  pdl_wait();
  const float* z = p.z + row * p.ld;
  const int shift = (int)((uintptr_t)z >> 2) & 3;        // logits before the row in its first 16 bytes
  const int vecs = (p.n + shift + 3) / 4, tiles = (vecs + kTile - 1) / kTile;
  const auto load = [&](int vec, float* v) {
    const int j = vec * 4 - shift;
    if (j >= 0 && j + 4 <= p.n) {
      const float4 q = __ldcs(reinterpret_cast<const float4*>(z + j));
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = j + e >= 0 && j + e < p.n ? z[j + e] : -INFINITY;
    }
  };
  const int mine = (tiles - part + p.parts - 1) / p.parts, per = (mine + kGroups - 1) / kGroups;      // this CTA's tiles, and those of a group
  LogStat s{-INFINITY, 0.f, 0.f};
  float in_group = -INFINITY;
  float next[4 * kVecs];      // the next tile's, on their way while a tile is added up (500 rows of 151936, us: 56 -> 52)
  const auto fetch = [&](int i) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) load((part + i * p.parts) * kTile + k * kThreads + threadIdx.x, next + 4 * k);
  };
  if (mine > 0) fetch(0);
  for (int i = 0, left = per, group = 0; i < mine; ++i) {
    float v[4 * kVecs];
#pragma unroll
    for (int k = 0; k < 4 * kVecs; ++k) v[k] = next[k];
    if (i + 1 < mine) fetch(i + 1);
    float largest = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4 * kVecs; ++k) largest = fmaxf(largest, v[k]);
    add_terms(s, v, largest);
    if (TOP) {
      in_group = fmaxf(in_group, largest);
      if (--left == 0 || i == mine - 1) {
        sh.group[group++][threadIdx.x] = in_group;
        in_group = -INFINITY;
        left = per;
      }
    }
  }

  unsigned long long list = 0;
  if (TOP) {
    if (threadIdx.x == 0) sh.count = 0;
    float best = sort_lanes(s.m, lane);
    sh.best[warp][lane] = best;
    __syncthreads();
#pragma unroll
    for (int half = kWarps / 2; half > 0; half >>= 1) {
      if (warp < half) {
        best = merge_floats(best, sh.best[warp + half][lane], lane);
        sh.best[warp][lane] = best;
      }
      __syncthreads();
    }
    const float bound = sh.best[0][p.top - 1];
    if (s.m >= bound && s.m > -INFINITY)
      for (int g = 0; g * per < mine; ++g) {
        const float x = sh.group[g][threadIdx.x];
        if (x >= bound && x > -INFINITY) sh.chosen[atomicAdd(&sh.count, 1)] = g * kThreads + threadIdx.x;      // (whatever their order, the same logits come out)
      }
    __syncthreads();
    // their vectors, dealt out to the warps one by one
    const int each = per * kVecs, items = sh.count * each;
    unsigned long long last = 0;
    for (int base = 0; base < items; base += kThreads) {
      const int q = base + lane * kWarps + warp;
      int id = p.n;
      float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (q < items) {
        const int what = sh.chosen[q / each], k = q % each, i = what / kThreads * per + k / kVecs;
        if (i < mine) {
          const int vec = (part + i * p.parts) * kTile + k % kVecs * kThreads + what % kThreads;
          load(vec, v);
          id = vec * 4 - shift;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) offer(list, last, v[e] >= bound && v[e] > -INFINITY ? logit_key(v[e], id + e) : 0, p.top, lane);
    }
  }

  // warps, then CTAs, into the first ones
  s = join_lanes<32>(s);
  if (lane == 0) sh.stat[warp] = s;
  if (TOP) sh.list[warp][lane] = list;
  __syncthreads();
  if (TOP) {
#pragma unroll
    for (int half = kWarps / 2; half > 0; half >>= 1) {
      if (warp < half) {
        list = merge_lists(list, sh.list[warp + half][lane], lane);
        sh.list[warp][lane] = list;
      }
      __syncthreads();
    }
  }
  if (p.parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (warp == 0) {
    s = join_lanes<kWarps>(sh.stat[lane % kWarps]);
    if (p.parts > 1) {
      const uint32_t at = map_cluster(smem_u32(&sh.parts[part]), 0);
      if (lane == 0)
        asm volatile("st.shared::cluster.f32 [%0], %1; st.shared::cluster.f32 [%0+4], %2; st.shared::cluster.f32 [%0+8], %3;" ::"r"(at), "f"(s.m),
                     "f"(s.s), "f"(s.t)
                     : "memory");
      if (TOP) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(map_cluster(smem_u32(&sh.part_list[part][lane]), 0)), "l"(list) : "memory");
    }
  }
  if (p.parts > 1) {
    __syncwarp();
    cluster_sync_all();
    if (part) return;
    if (warp == 0) {
      const bool there = lane < p.parts;
      s = join_lanes<32>(there ? sh.parts[lane] : LogStat{-INFINITY, 0.f, 0.f});
    }
    if (TOP) {
      for (int half = p.parts / 2; half > 0; half >>= 1) {
        if (warp < half) sh.part_list[warp][lane] = merge_lists(sh.part_list[warp][lane], sh.part_list[warp + half][lane], lane);
        __syncthreads();
      }
      list = sh.part_list[0][lane];
    }
  }
  if (warp) return;
  const LogNorm norm = log_norm(s);
  if (lane == 0) {
    const int t = p.tokens[row];
    p.logprob[row] = t >= 0 && t < p.n ? log_prob(norm, z[t]) : NAN;
    p.entropy[row] = norm.entropy;
  }
  if (TOP) {
    list = fill_list(list, z, p.n, p.top, lane);
    if (lane < p.top) {
      p.top_ids[(long long)row * p.top + lane] = list ? (int)key_id(list) : -1;
      p.top_logprobs[(long long)row * p.top + lane] = list ? log_prob(norm, order_value((uint32_t)(list >> 32))) : -INFINITY;
    }
  }
}

int sm_count() {
  static int n[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!n[dev & 63]) cudaDeviceGetAttribute(&n[dev & 63], cudaDevAttrMultiProcessorCount, dev);
  return n[dev & 63];
}

template <bool TOP>
int launch(const RowsParams& p, int m, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(logprob_rows_kernel<TOP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return (int)e;
    configured[dev & 63] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)m * p.parts);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (p.parts > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = p.parts;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (!b2_no_pdl()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return (int)cudaLaunchKernelEx(&cfg, logprob_rows_kernel<TOP>, p);
}

}  // namespace

// z: [m] rows of n logits, ld elements apart.  top: alternatives per row, at most kMaxTop.
extern "C" int b2_logprob_rows(const float* z, long long ld, int m, int n, const int* tokens, int top, float* logprob, float* entropy,
                               int* top_ids, float* top_logprobs, void* stream) {
  if (m < 1 || n < 1 || n > 0x7fff0000 || ld < n || top < 0 || top > kMaxTop || ((uintptr_t)z & 3)) return -1;
  // CTAs of a row: as many as it has tiles, and as leave four to an SM; sixteen, whose joining costs most, where there are two to an SM.
  // Rows of 151936, 10 alternatives, us with 1 / 2 / 4 / 8 / 16 CTAs a row (an earlier form): 8 rows 27.4 / 16.5 / 11.2 / 8.1 / 7.9, 32 rows 27.6 / 16.6 /
  // 11.5 / 9.7 / 14.3, 100 rows 41.8 / 26.8 / 19.0 / 23.0 / 34.2, 200 rows 49.7 / 32.6 / 37.9 / 39.2 / 63.6, 500 rows 65.8 / 67.5 / 78.4 / 94.8 / 153.4.
  // What the rule does not see is how many SMs get one CTA more than the others: 297 to 400 rows have a CTA each, some SMs three of them, and take 39
  // to 42 us whatever their number (27.5 to 37 of bytes).
  const int tiles = ((n + 6) / 4 + kTile - 1) / kTile, sms = sm_count();
  int parts = 1;
  while (parts < kParts && 2 * parts <= tiles && 2ll * parts * m <= (2 * parts == kParts ? 2 : 4) * sms) parts *= 2;
  const RowsParams p{z, ld, n, top, parts, tokens, logprob, entropy, top_ids, top_logprobs};
  return top ? launch<true>(p, m, (cudaStream_t)stream) : launch<false>(p, m, (cudaStream_t)stream);
}

B2_DEFINE_STATUS(logprob)
