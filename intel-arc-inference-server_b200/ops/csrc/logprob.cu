// Log probabilities of given tokens, entropy and top alternatives of rows of fp32 logits.
//
//   d_j = z_j - max z      S = sum_j exp d_j      log p_t = d_t - ln S      H = ln S - (sum_j d_j exp d_j) / S
//
// One pass over a row: its logits go through registers once, each thread with a maximum and sums of its own (LogStat).  A cluster of up
// to 16 CTAs shares a row and joins its results in the first CTA's shared memory: no workspace, no counters, the same order of every sum
// in every run.
//
// Alternatives: the top-th largest of the threads' maxima is a bound that at least `top` logits of the CTA reach, so only the logits of the
// threads whose maximum reaches it can matter: about `top` threads of a CTA.  Those few are read again, and what reaches the bound is put
// in order.  The pass itself does nothing for the alternatives.
#include "common.cuh"
#include "logprob.cuh"
#include "pair.cuh"

using namespace b2;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kVecs = 4;                              // 16-byte vectors of a thread and tile
constexpr int kTile = kThreads * kVecs;               // vectors
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

struct Shared {
  LogStat stat[kWarps], parts[kParts];
  unsigned long long list[kWarps][32], part_list[kParts][32];
  float best[kWarps][32];
  int chosen, threads[kThreads];
};

__device__ __forceinline__ uint32_t map_cluster(uint32_t addr, int rank) {      // a CTA's copy of a shared-memory word
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

template <bool TOP>
__global__ void __launch_bounds__(kThreads, 5) logprob_rows_kernel(const RowsParams p) {
  __shared__ Shared sh;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (p.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // the first CTA is there: waited for below
  pdl_wait();
  const float* z = p.z + row * p.ld;
  const int shift = (int)((uintptr_t)z >> 2) & 3;        // logits before the row in its first 16 bytes
  const int vecs = (p.n + shift + 3) / 4, tiles = (vecs + kTile - 1) / kTile;
  const auto load = [&](int tile, float (&v)[4 * kVecs]) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int vec = tile * kTile + i * kThreads + threadIdx.x, j = vec * 4 - shift;
      if (j >= 0 && j + 4 <= p.n) {
        const float4 q = __ldcs(reinterpret_cast<const float4*>(z + j));
        v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * i + e] = j + e >= 0 && j + e < p.n ? z[j + e] : -INFINITY;
      }
    }
  };
  LogStat s{-INFINITY, 0.f, 0.f};
  for (int tile = part; tile < tiles; tile += p.parts) {
    float v[4 * kVecs];
    load(tile, v);
    float largest = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * kVecs; ++i) largest = fmaxf(largest, v[i]);
    add_terms(s, v, largest);
  }

  unsigned long long list = 0;
  if (TOP) {
    const float mine = s.m;
    if (threadIdx.x == 0) sh.chosen = 0;
    float best = sort_lanes(mine, lane);
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
    const bool choose = mine >= bound && mine > -INFINITY;
    const uint32_t mask = __ballot_sync(0xffffffffu, choose);
    int at = 0;
    if (lane == 0 && mask) at = atomicAdd(&sh.chosen, __popc(mask));      // (whatever their order, the same logits come out)
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(mask & ((1u << lane) - 1));
    if (choose) sh.threads[at] = threadIdx.x;
    __syncthreads();
    // the chosen threads' vectors, dealt out to the warps one by one
    const int each = (tiles - part + p.parts - 1) / p.parts * kVecs, items = sh.chosen * each;
    unsigned long long last = 0;
    for (int base = 0; base < items; base += kThreads) {
      const int q = base + lane * kWarps + warp;
      int id = p.n;
      float v[4];
      if (q < items) {
        const int thread = sh.threads[q / each], i = q % each, vec = (part + i / kVecs * p.parts) * kTile + i % kVecs * kThreads + thread;
        id = vec * 4 - shift;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = id + e >= 0 && id + e < p.n ? z[id + e] : -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned long long key = v[e] >= bound && v[e] > -INFINITY ? logit_key(v[e], id + e) : 0;
        uint32_t more = __ballot_sync(0xffffffffu, key > last);
        while (more) {
          insert(list, __shfl_sync(0xffffffffu, key, __ffs(more) - 1), lane);
          last = __shfl_sync(0xffffffffu, list, p.top - 1);
          more = __ballot_sync(0xffffffffu, key > last) & (more & (more - 1));
        }
      }
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
    // Fewer than `top` logits above -inf: banned ids follow, the lowest first, then those without a number.
    int have = __popc(__ballot_sync(0xffffffffu, list != 0));
    for (int kind = 0; kind < 2 && have < p.top; ++kind) {
      for (int j0 = 0; j0 < p.n && have < p.top; j0 += 32) {
        const int j = j0 + lane;
        const float x = j < p.n ? z[j] : 0.f;
        const bool take = j < p.n && (kind == 0 ? x == -INFINITY : x != x);
        const uint32_t mask = __ballot_sync(0xffffffffu, take);
        const int nth = lane - have;      // this lane's place is the nth of them
        if (nth >= 0 && nth < __popc(mask)) {
          const int from = __fns(mask, 0, nth + 1);
          list = logit_key(kind == 0 ? -INFINITY : __int_as_float(0x7fffffff), j0 + from);
        }
        have += __popc(mask);
      }
    }
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
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.parts > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, logprob_rows_kernel<TOP>, p);
}

}  // namespace

// z: [m] rows of n logits, ld elements apart.  top: alternatives per row, at most kMaxTop.
extern "C" int b2_logprob_rows(const float* z, long long ld, int m, int n, const int* tokens, int top, float* logprob, float* entropy,
                               int* top_ids, float* top_logprobs, void* stream) {
  if (m < 1 || n < 1 || n > 0x7fff0000 || ld < n || top < 0 || top > kMaxTop || ((uintptr_t)z & 3)) return -1;
  // CTAs of a row: as many as it has tiles, and as leave four to an SM; sixteen, whose joining costs most, where there are two to an SM.
  // Rows of 151936, 10 alternatives, 1 / 2 / 4 / 8 / 16 CTAs a row, us: 8 rows 27.4 / 16.5 / 11.2 / 8.1 / 7.9, 32 rows 27.6 / 16.6 / 11.5 / 9.7 / 14.3,
  // 100 rows 41.8 / 26.8 / 19.0 / 23.0 / 34.2, 200 rows 49.7 / 32.6 / 37.9 / 39.2 / 63.6, 500 rows 65.8 / 67.5 / 78.4 / 94.8 / 153.4.
  const int tiles = ((n + 6) / 4 + kTile - 1) / kTile, sms = sm_count();
  int parts = 1;
  while (parts < kParts && 2 * parts <= tiles && 2ll * parts * m <= (2 * parts == kParts ? 2 : 4) * sms) parts *= 2;
  const RowsParams p{z, ld, n, top, parts, tokens, logprob, entropy, top_ids, top_logprobs};
  return top ? launch<true>(p, m, (cudaStream_t)stream) : launch<false>(p, m, (cudaStream_t)stream);
}
extern "C" int b2_logprob_max_top() { return kMaxTop; }

B2_DEFINE_STATUS(logprob)
