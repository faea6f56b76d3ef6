// A prompt's rows through the head: z = x W^T (bf16), or (q . w) s_row s_column (int8), on tcgen05, two SMs on one 256 x 256 tile.  The
// logits of a tile leave tensor memory for registers and go no further: what stays of 256 logits of a row are their maximum and two sums
// (LogStat, 16 bytes in place of 1024), and the token's logit where it is among them.  A second kernel joins a row's tiles in order.
// With alternatives the logits themselves are stored, for logprob.cu.
//
// Structure, per cluster of two CTAs (192 threads each):
//   warp 0    copies by TMA: this CTA's 128 rows of x and 128 of the tile's 256 rows of W, 128 bytes of k a stage, six stages
//   warp 1    even CTA: tcgen05.mma.cta_group::2, M = 256, N = 256; two accumulators in tensor memory
//   warps 2-5 this CTA's 128 rows of the accumulator, a thread per row: sums, or logits to memory
// Tiles are walked rows first, so that the clusters that run together share the rows of W in L2.
#include "common.cuh"
#include "logprob.cuh"
#include "pair.cuh"

using namespace b2;

namespace {

constexpr int BM = 128, BN = 256, kStageRow = 128;      // rows of a CTA, columns of a tile, bytes of k a stage
constexpr int kThreads = 192;
constexpr int kHalf = 128 * kStageRow, kStage = 2 * kHalf, kStages = 6;
constexpr int kSmem = kStages * kStage + 1024 + 256;    // + alignment, barriers

struct ScoreParams {
  int m, n, kb;             // kb: stages of k
  const float *x_scale, *w_scale;      // int8: per row of x, per row of W
  float* z;                 // [m][ldz] logits
  long long ldz;
  const int* tokens;        // sums: [m]
  float4* part;             // [column of tiles][m]: maximum and sums of a row's 256 logits
  float* token_z;           // [m] logit of the row's token, where it has one
};

__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// SUMS: maxima and sums; else logits.
template <bool I8, bool SUMS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
score_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const ScoreParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ float scales[2][I8 ? BN : 1];      // of the columns of a tile and of the next
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u, bars = smem + kStages * kStage;
  const uint32_t full0 = bars, empty0 = full0 + 8 * kStages, done0 = empty0 + 8 * kStages, read0 = done0 + 16, slot = read0 + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_rank();
  const int tiles_m = (p.m + 2 * BM - 1) / (2 * BM), tiles = tiles_m * ((p.n + BN - 1) / BN);
  const int first = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full0 + 8 * i, 1);      // used in the even CTA: both CTAs' bytes
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(done0 + 8 * i, 1);
      mbar_init(read0 + 8 * i, 8);      // used in the even CTA: both CTAs' four warps
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();      // both CTAs' barriers are there before anything arrives on them
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&map_x);
      prefetch_tmap(&map_w);
      int s = 0, round = 0, issued = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += pairs) {
        const int row0 = (t % tiles_m) * 2 * BM + rank * BM, col0 = (t / tiles_m) * BN + rank * (BN / 2);
        for (int kb = 0; kb < p.kb; ++kb) {
          if (round > 0) ok = mbar_wait_lone(empty0 + 8 * s, (round - 1) & 1, ERR_GEMM_EMPTY_WAIT);
          if (!ok) break;
          const uint32_t at = smem + s * kStage, bar = map_rank0(full0 + 8 * s);
          if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * kStage);
          tma_load_2d_pair(at, &map_x, kb * (I8 ? kStageRow : kStageRow / 2), row0, bar);
          tma_load_2d_pair(at + kHalf, &map_w, kb * (I8 ? kStageRow : kStageRow / 2), col0, bar);
          ++issued;
          if (++s == kStages) { s = 0; ++round; }
        }
      }
      // After a wait that ran out the even CTA waits (bounded) for the bytes both have asked for; the odd one meets it at the cluster
      // barrier below.
      if (!ok && rank == 0)
        for (int i = max(0, issued - kStages); i < issued; ++i) mbar_wait(full0 + 8 * (i % kStages), (i / kStages) & 1, ERR_GEMM_FULL_WAIT);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = I8 ? make_idesc(2, 1, 2 * BM, BN) : make_idesc(1, 1, 2 * BM, BN);
      int s = 0, par = 0, i = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += pairs, ++i) {
        const int a = i & 1;
        if (i >= 2) ok = mbar_wait_cluster(read0 + 8 * a, ((i >> 1) - 1) & 1, ERR_GEMM_TMEM_EMPTY_WAIT);
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < p.kb; ++kb) {
          ok = mbar_wait_cluster(full0 + 8 * s, par, ERR_GEMM_FULL_WAIT);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = make_desc_sw128(smem + s * kStage), db = make_desc_sw128(smem + s * kStage + kHalf);
#pragma unroll
          for (int k = 0; k < 4; ++k) {      // 32 bytes of k each
            if (I8) umma_i8_pair(tmem + a * BN, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
            else umma_f16_pair(tmem + a * BN, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
          }
          tc_commit_pair(empty0 + 8 * s);
          if (++s == kStages) { s = 0; par ^= 1; }
        }
        if (ok) tc_commit_pair(done0 + 8 * a);
      }
    }
  } else {
    const int quarter = warp & 3;      // of the lanes of tensor memory, this warp's
    int i = 0;
    bool ok = true;
    for (int t = first; t < tiles; t += pairs, ++i) {      // (to the end also after a wait that ran out: the warps meet at a barrier)
      const int a = i & 1, row0 = (t % tiles_m) * 2 * BM + rank * BM + quarter * 32, row = row0 + lane, nt = t / tiles_m, col0 = nt * BN;
      if (I8) {      // (written while others may still read the tile before: two buffers)
        const int j = threadIdx.x - 64;
        scales[a][j] = p.w_scale[min(col0 + j, p.n - 1)];
        scales[a][j + 128] = p.w_scale[min(col0 + j + 128, p.n - 1)];
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      const bool there = row < p.m;
      const float xs = I8 && there ? p.x_scale[row] : 1.f;
      const int token = SUMS && there ? p.tokens[row] : -1;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(done0 + 8 * a, (i >> 1) & 1, ERR_GEMM_TMEM_FULL_WAIT));
      if (!ok) continue;
      tc_fence_after();
      LogStat s{-INFINITY, 0.f, 0.f};
#pragma unroll 1
      for (int c = 0; c < BN / 32 && row0 < p.m; ++c) {
        uint32_t v[32];
        B2_TMEM_LD_32(tmem + a * BN + c * 32 + ((uint32_t)(quarter * 32) << 16), v);
        tmem_ld_wait();
        const int n0 = col0 + c * 32;
        if (n0 >= p.n) break;
        if (I8) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint((float)(int)v[j] * xs * scales[a][c * 32 + j]);
        }
        if (SUMS) {
          float z[32], largest = -INFINITY;
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] = __uint_as_float(v[j]);
          if (n0 + 32 > p.n) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (n0 + j >= p.n) z[j] = -INFINITY;
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) largest = fmaxf(largest, z[j]);
          add_terms(s, z, largest);
          if (token >= n0 && token < min(n0 + 32, p.n)) {
            float mine = z[0];
#pragma unroll
            for (int j = 1; j < 32; ++j) mine = token == n0 + j ? z[j] : mine;
            p.token_z[row] = mine;
          }
        } else if (there) {
          float* dst = p.z + row * p.ldz + n0;
          if (n0 + 32 <= p.n) {
#pragma unroll
            for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(dst + 4 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (n0 + j < p.n) dst[j] = __uint_as_float(v[j]);
          }
        }
      }
      if (SUMS && there) p.part[(long long)nt * p.m + row] = make_float4(s.m, s.s, s.t, 0.f);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_rank0(read0 + 8 * a));
    }
  }

  // every thread of both CTAs arrives here on every path
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ------------------------------------------------------------------ a row's tiles together
// A CTA takes 32 rows: warp w joins tiles w, w + 32, ... of all of them (a lane a row, so that a warp reads whole lines), then the warps'
// results are joined in the order of the warps.
__global__ void __launch_bounds__(1024) score_join_kernel(const float4* __restrict__ part, const float* __restrict__ token_z, const int* __restrict__ tokens, int m,
                                                          int n, float* __restrict__ logprob, float* __restrict__ entropy) {
  __shared__ LogStat sh[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * 32 + lane, tiles = (n + BN - 1) / BN;
  pdl_wait();
  LogStat s{-INFINITY, 0.f, 0.f};
  if (row < m)
#pragma unroll 4
    for (int t = warp; t < tiles; t += 32) {
      const float4 q = part[(long long)t * m + row];
      s = join(s, LogStat{q.x, q.y, q.z});
    }
  sh[warp][lane] = s;
  __syncthreads();
#pragma unroll
  for (int half = 16; half > 0; half >>= 1) {
    if (warp < half) sh[warp][lane] = s = join(s, sh[warp + half][lane]);
    __syncthreads();
  }
  if (warp == 0 && row < m) {
    const LogNorm norm = log_norm(s);
    const int t = tokens[row];
    logprob[row] = t >= 0 && t < n ? log_prob(norm, token_z[row]) : NAN;
    entropy[row] = norm.entropy;
  }
}

// ------------------------------------------------------------------ rows as int8 with a scale per row
// s = max|x| / 127, q = rint(x (1 / s)): 8 bits a value, off by at most s / 2.  A row with a NaN or an infinity has the scale NaN, and so
// have its logits; no scale is below 2^-126, whose inverse is finite.  One CTA per row, 16 bytes a thread and step.
__global__ void __launch_bounds__(256) quant_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, int k, int8_t* __restrict__ q, long long ldq,
                                                    float* __restrict__ scale) {
  __shared__ float part[8];
  const uint4* row = reinterpret_cast<const uint4*>(x + blockIdx.x * ldx);
  const int vecs = k / 8, tail = k % 8;
  const __nv_bfloat16* end = x + blockIdx.x * ldx + vecs * 8;
  float largest = 0.f;
  for (int i = threadIdx.x; i < vecs; i += 256) {
    const uint4 v = __ldg(row + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) largest = max_nan(largest, max_nan(fabsf(bf16_lo(w[j])), fabsf(bf16_hi(w[j]))));
  }
  if (threadIdx.x < tail) largest = max_nan(largest, fabsf(__bfloat162float(end[threadIdx.x])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = largest;
  __syncthreads();
  largest = part[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) largest = max_nan(largest, part[i]);
  const bool finite = largest < INFINITY;
  const float s = fmaxf(largest / 127.f, 1.17549435e-38f), inv = finite ? 1.f / s : 0.f;
  int8_t* out = q + blockIdx.x * ldq;
  for (int i = threadIdx.x; i < vecs; i += 256) {
    const uint4 v = __ldg(row + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[j >> 1] |= (uint32_t)(__float2int_rn(bf16_lo(w[j]) * inv) & 0xff) << (16 * (j & 1));
      o[j >> 1] |= (uint32_t)(__float2int_rn(bf16_hi(w[j]) * inv) & 0xff) << (16 * (j & 1) + 8);
    }
    reinterpret_cast<uint2*>(out)[i] = make_uint2(o[0], o[1]);
  }
  if (threadIdx.x < tail) out[vecs * 8 + threadIdx.x] = (int8_t)__float2int_rn(__bfloat162float(end[threadIdx.x]) * inv);
  if (threadIdx.x == 0) scale[blockIdx.x] = finite ? s : NAN;
}

// ------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  return fn;
}

// 128 rows x 128 bytes of a matrix [rows][cols], rows ld elements apart; what lies outside reads as zeros
int make_map(CUtensorMap* map, const void* ptr, bool i8, int rows, int cols, long long ld) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return -100;
  const int size = i8 ? 1 : 2;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * size};
  const cuuint32_t box[2] = {(cuuint32_t)(kStageRow / size), 128}, step[2] = {1, 1};
  const CUresult r = fn(map, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -101 - (int)r;
}

int sm_count() {
  static int n[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!n[dev & 63]) cudaDeviceGetAttribute(&n[dev & 63], cudaDevAttrMultiProcessorCount, dev);
  return n[dev & 63];
}

template <bool I8, bool SUMS>
int launch(const CUtensorMap& mx, const CUtensorMap& mw, const ScoreParams& p, int tiles, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(score_kernel<I8, SUMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return (int)e;
    configured[dev & 63] = true;
  }
  score_kernel<I8, SUMS><<<2 * min(tiles, sm_count() / 2), kThreads, kSmem, st>>>(mx, mw, p);
  return (int)cudaGetLastError();
}

int run(const void* x, long long ldx, const void* w, long long ldw, bool i8, int k, ScoreParams& p, bool sums, cudaStream_t st) {
  const int size = i8 ? 1 : 2;
  const long long tiles = (long long)((p.m + 2 * BM - 1) / (2 * BM)) * ((p.n + BN - 1) / BN);
  if (p.m < 1 || p.n < 1 || (long long)k * size < kStageRow || ldx < k || ldw < k || tiles > 0x3fffffff || (i8 && (!p.x_scale || !p.w_scale))) return -1;
  if (((uintptr_t)x | (uintptr_t)w | (unsigned long long)(ldx * size) | (unsigned long long)(ldw * size)) & 15) return -3;
  p.kb = (int)(((long long)k * size + kStageRow - 1) / kStageRow);
  CUtensorMap mx, mw;
  int rc = make_map(&mx, x, i8, p.m, k, ldx);
  if (!rc) rc = make_map(&mw, w, i8, p.n, k, ldw);
  if (rc) return rc;
  if (sums) return i8 ? launch<true, true>(mx, mw, p, (int)tiles, st) : launch<false, true>(mx, mw, p, (int)tiles, st);
  return i8 ? launch<true, false>(mx, mw, p, (int)tiles, st) : launch<false, false>(mx, mw, p, (int)tiles, st);
}

}  // namespace

// Rows x [m][k] against the head w [n][k], both bf16, or int8 with scales; rows are ldx and ldw elements apart, multiples of 16 bytes, of
// 128 bytes at least.
// Logits z [m][ldz], ldz a multiple of 4.
extern "C" int b2_score_logits(const void* x, long long ldx, const void* w, long long ldw, int i8, const float* x_scale, const float* w_scale, int m, int n,
                               int k, float* z, long long ldz, void* stream) {
  if (ldz < n || (((uintptr_t)z | (unsigned long long)(ldz * 4)) & 15)) return -2;
  ScoreParams p{m, n, 0, x_scale, w_scale, z, ldz, nullptr, nullptr, nullptr};
  return run(x, ldx, w, ldw, i8 != 0, k, p, false, (cudaStream_t)stream);
}
// Log probabilities of the rows' tokens and entropies.  work: b2_score_work(m, n) floats, 16-byte aligned, of this call alone.
extern "C" long long b2_score_work(int m, int n) { return ((long long)((n + BN - 1) / BN) * 4 + 1) * m; }
extern "C" int b2_score_tokens(const void* x, long long ldx, const void* w, long long ldw, int i8, const float* x_scale, const float* w_scale, int m, int n,
                               int k, const int* tokens, float* work, float* logprob, float* entropy, void* stream) {
  if ((uintptr_t)work & 15) return -2;
  float* token_z = work + (long long)((n + BN - 1) / BN) * 4 * m;
  ScoreParams p{m, n, 0, x_scale, w_scale, nullptr, 0, tokens, (float4*)work, token_z};
  const int rc = run(x, ldx, w, ldw, i8 != 0, k, p, true, (cudaStream_t)stream);
  if (rc) return rc;
  return b2_launch(score_join_kernel, dim3((m + 31) / 32), dim3(1024), 0, (cudaStream_t)stream, true, (const float4*)work, token_z, tokens, m, n, logprob, entropy);
}

// Rows x [m][k] bf16 (16-byte aligned, ldx a multiple of 8) as int8 q [m][ldq] (16-byte aligned, ldq a multiple of 16) and scales.
extern "C" int b2_score_quant(const void* x, long long ldx, int m, int k, void* q, long long ldq, float* scale, void* stream) {
  if (m < 1 || k < 1 || ldx < k || ldq < k || ((uintptr_t)x | (uintptr_t)q | (unsigned long long)(ldx * 2) | (unsigned long long)ldq) & 15) return -1;
  quant_kernel<<<m, 256, 0, (cudaStream_t)stream>>>((const __nv_bfloat16*)x, ldx, k, (int8_t*)q, ldq, scale);
  return (int)cudaGetLastError();
}

B2_DEFINE_STATUS(score)
