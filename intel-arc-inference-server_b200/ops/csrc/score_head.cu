// A prompt's rows through the head: z = x W^T (bf16), or (q . w) s_row s_column (int8), on tcgen05.  The logits of a tile leave tensor memory
// for registers: what stays of a row's logits there are their maximum and two sums (LogStat), and the token's logit where it is among
// them.  A second kernel joins a row's parts in order.  With alternatives the logits are stored too, beside the largest of every 32; the
// second kernel reads these maxima and only those logits whose maximum reaches the top-th largest of a few (as in logprob.cu).
//
// Two forms.  PAIR: a cluster of two CTAs on a 256 x 256 tile (tcgen05 cta_group::2), which asks least of the L2.  Else a CTA by itself on 128 x
// 256, for up to 128 rows, where the head's bytes are what counts and the multiplication has to keep out of their way, and for 257 to 384,
// of which pairs would multiply 512.  Pairs / CTAs by themselves, us, 151936 x 5120: 64 rows 297 / 271, 256 rows 324 / 352, 300 rows
// 528 / 466, 512 rows 565 / 618.
//   warp 0    copies by TMA: 128 rows of x and the CTA's rows of the tile of W (128 or 256), 128 bytes of k a stage
//   warp 1    tcgen05.mma (PAIR: of the even CTA), N = 256; two accumulators in tensor memory
//   warps 2-5 the CTA's 128 rows of the accumulator, a thread per row
// More than 512 rows: tiles are walked rows first, so that the clusters that run together share the rows of W in L2.  Up to 512 rows whole
// tiles would leave SMs idle at the end (102400 columns: 400 tiles for 74 clusters): every cluster gets a range of columns of its own,
// equal but for 32, whose last tile is as narrow as it has to be; a thread's sums go on through the range.
//
// More than about 300 rows are bound by the multiplication: 4096 rows x 151936 x 5120 take 3.6 ms in a short run (1.78 PFLOP/s) and 4.1 under
// the power cap, int8 1.86 and 2.2 ms; halving the copies of x changes nothing, four warps more for the sums cost 5 %.  Fewer rows are
// bound by the head's bytes: 77 rows x 102400 x 2048 72 us (5.8 TB/s), 64 rows x 151936 x 5120 260 us with the join (6.0 TB/s).  With
// the logits stored and read again by logprob.cu (with alternatives it was so once) 900 rows x 151936 x 5120 took 1.41 ms, now 1.20.
#include "common.cuh"
#include "logprob.cuh"
#include "pair.cuh"

using namespace b2;

namespace {

constexpr int BM = 128, BN = 256, kStageRow = 128;      // rows of a CTA, columns of a tile, bytes of k a stage
constexpr int kThreads = 192;
constexpr int kGrain = 32, kChunk = 32;        // columns that ranges are cut at, columns of a maximum
constexpr int kMostI8 = 1 << 17;       // columns of 127 x 127 that an int32 sum holds
constexpr int kRangeRows = 512;      // up to these many rows ranges

template <bool PAIR>
struct Form {
  static constexpr int ROWS = PAIR ? 2 * BM : BM;                   // of a tile
  static constexpr int X_BYTES = BM * kStageRow, W_BYTES = (PAIR ? BN / 2 : BN) * kStageRow, STAGE = X_BYTES + W_BYTES;
  static constexpr int STAGES = PAIR ? 6 : 4;
  static constexpr int SMEM = STAGES * STAGE + 1024 + 256;          // + alignment, barriers
};
constexpr int kOutBytes = BM * kChunk * 4;      // alternatives: the warps' 32 x 32 logits on their way out

struct ScoreParams {
  int m, n, kb;             // kb: stages of k
  int ranges;               // of columns, for each row of tiles; 0: tiles in turn
  const float *x_scale, *w_scale;      // int8: per row of x, per row of W
  const int* tokens;        // [m]
  float4* part;             // [range, or column of tiles][m]: maximum and sums of a row's logits
  float* token_z;           // [m] logit of the row's token, where it has one
  float* largest;           // alternatives: the largest of every kChunk logits [m][ldc]
  int ldc;
};

__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The tiles of a cluster, one after another: row of tiles mt, columns [col0, end) of which the tile has `width`, a multiple of 32; part: where
// its sums go.
struct Tile {
  int mt, col0, end, width, part;
};
template <bool PAIR>
__device__ __forceinline__ bool tile_at(const ScoreParams& p, int i, Tile& t) {
  const int first = PAIR ? blockIdx.x >> 1 : blockIdx.x, tiles_m = (p.m + Form<PAIR>::ROWS - 1) / Form<PAIR>::ROWS;
  if (p.ranges) {
    const long long grains = (p.n + kGrain - 1) / kGrain;
    t.mt = first % tiles_m;
    t.part = first / tiles_m;
    t.col0 = (int)(t.part * grains / p.ranges) * kGrain + i * BN;
    t.end = min(p.n, (int)((t.part + 1) * grains / p.ranges) * kGrain);
    t.width = min(BN, (t.end - t.col0 + kGrain - 1) / kGrain * kGrain);
    return t.col0 < t.end;
  }
  const int at = first + i * (PAIR ? gridDim.x >> 1 : gridDim.x);
  t.mt = at % tiles_m;
  t.part = at / tiles_m;
  t.col0 = t.part * BN;
  t.end = p.n;
  t.width = BN;
  return t.col0 < p.n;
}

// Rows of x that a CTA fetches of a block of 128 that begins at row0: those that there are, in eights.  (Rows outside the matrix cost a copy more than
// rows inside: with boxes of 128 for all, 1 row x 102400 x 2048 took 100 us, 16 rows 87, 77 rows 76; with these 74 to 76.)  What the rest
// of the block holds then goes to rows of the accumulator that nobody reads.
__device__ __forceinline__ int rows_at(const ScoreParams& p, int row0) { return min(BM, max(0, (p.m - row0 + 7) / 8 * 8)); }

// ALT: logits (map_z, 32 x 32 at a time) and their maxima are stored.  map_e: the rows behind the last whole block of 128 of x; map_g: W in boxes of 16 (PAIR) or 32
// rows, for narrow tiles.
template <bool I8, bool ALT, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
score_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_e, const __grid_constant__ CUtensorMap map_w,
             const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_z, const ScoreParams p) {
  using F = Form<PAIR>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ float scales[2][I8 ? BN : 1];      // of the columns of a tile and of the next
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u, bars = smem + F::STAGES * F::STAGE + (ALT ? kOutBytes : 0);
  const uint32_t full0 = bars, empty0 = full0 + 8 * F::STAGES, done0 = empty0 + 8 * F::STAGES, read0 = done0 + 16, slot = read0 + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = PAIR ? (int)cluster_rank() : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < F::STAGES; ++i) {
      mbar_init(full0 + 8 * i, 1);      // PAIR: used in the even CTA, both CTAs' bytes
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(done0 + 8 * i, 1);
      mbar_init(read0 + 8 * i, PAIR ? 8 : 4);      // PAIR: used in the even CTA, both CTAs' four warps
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(slot, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();      // both CTAs' barriers are there before anything arrives on them
  tc_fence_after();
  pdl_wait();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&map_x);
      prefetch_tmap(&map_w);
      int s = 0, round = 0, issued = 0;
      bool ok = true;
      Tile t;
      for (int i = 0; ok && tile_at<PAIR>(p, i, t); ++i) {
        const int row0 = t.mt * F::ROWS + rank * BM, mine = PAIR ? t.width / 2 : t.width, col0 = t.col0 + rank * mine;
        const int rows = rows_at(p, row0);
        const CUtensorMap* const map = rows == BM ? &map_x : &map_e;
        const uint32_t bytes = PAIR ? (rows + rows_at(p, row0 + BM) + 2 * mine) * kStageRow : (rows + mine) * kStageRow;      // (of the even CTA: both CTAs')
        for (int kb = 0; kb < p.kb; ++kb) {
          if (round > 0) ok = mbar_wait_lone(empty0 + 8 * s, (round - 1) & 1, ERR_GEMM_EMPTY_WAIT);
          if (!ok) break;
          const uint32_t at = smem + s * F::STAGE;
          const int k = kb * (I8 ? kStageRow : kStageRow / 2);
          if (PAIR) {
            const uint32_t bar = map_rank0(full0 + 8 * s);
            if (rank == 0) mbar_expect_tx(full0 + 8 * s, bytes);
            if (rows) tma_load_2d_pair(at, map, k, row0, bar);
            if (t.width == BN) tma_load_2d_pair(at + F::X_BYTES, &map_w, k, col0, bar);
            else
              for (int j = 0; j < mine; j += kGrain / 2) tma_load_2d_pair(at + F::X_BYTES + j * kStageRow, &map_g, k, col0 + j, bar);
          } else {
            const uint32_t bar = full0 + 8 * s;
            mbar_expect_tx(bar, bytes);
            tma_load_2d(at, map, k, row0, bar);
            if (t.width == BN) tma_load_2d(at + F::X_BYTES, &map_w, k, col0, bar);
            else
              for (int j = 0; j < mine; j += kGrain) tma_load_2d(at + F::X_BYTES + j * kStageRow, &map_g, k, col0 + j, bar);
          }
          ++issued;
          if (++s == F::STAGES) { s = 0; ++round; }
        }
      }
      // After a wait that ran out the (even) CTA waits (bounded) for the bytes that were asked for; the odd one meets it at the cluster
      // barrier below.
      if (!ok && rank == 0)
        for (int i = max(0, issued - F::STAGES); i < issued; ++i) mbar_wait(full0 + 8 * (i % F::STAGES), (i / F::STAGES) & 1, ERR_GEMM_FULL_WAIT);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int s = 0, par = 0;
      bool ok = true;
      Tile t;
      const auto wait = [](uint32_t bar, uint32_t parity, unsigned code) {
        return PAIR ? mbar_wait_cluster(bar, parity, code) : mbar_wait_lone(bar, parity, code);
      };
      const auto commit = [](uint32_t bar) {
        if (PAIR) tc_commit_pair(bar);
        else tc_commit(bar);
      };
      for (int i = 0; ok && tile_at<PAIR>(p, i, t); ++i) {
        const int a = i & 1;
        const uint32_t idesc = I8 ? make_idesc(2, 1, F::ROWS, t.width) : make_idesc(1, 1, F::ROWS, t.width);
        if (i >= 2) ok = wait(read0 + 8 * a, ((i >> 1) - 1) & 1, ERR_GEMM_TMEM_EMPTY_WAIT);
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < p.kb; ++kb) {
          ok = wait(full0 + 8 * s, par, ERR_GEMM_FULL_WAIT);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = make_desc_sw128(smem + s * F::STAGE), db = make_desc_sw128(smem + s * F::STAGE + F::X_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k) {      // 32 bytes of k each
            if (PAIR && I8) umma_i8_pair(tmem + a * BN, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
            else if (PAIR) umma_f16_pair(tmem + a * BN, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
            else if (I8) umma_i8(tmem + a * BN, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
            else umma_f16(tmem + a * BN, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
          }
          commit(empty0 + 8 * s);
          if (++s == F::STAGES) { s = 0; par ^= 1; }
        }
        if (ok) commit(done0 + 8 * a);
      }
    }
  } else {
    const int quarter = warp & 3;      // of the lanes of tensor memory, this warp's
    const uint32_t out = smem + F::STAGES * F::STAGE + quarter * (kOutBytes / 4);      // (a multiple of 1024; the barriers are behind it)
    bool ok = true;
    Tile t;
    LogStat s{-INFINITY, 0.f, 0.f};
    for (int i = 0; tile_at<PAIR>(p, i, t); ++i) {      // (to the end also after a wait that ran out: the warps meet at a barrier)
      const int a = i & 1, row0 = t.mt * F::ROWS + rank * BM + quarter * 32, row = row0 + lane;
      if (I8) {      // (written while others may still read the tile before: two buffers)
        const int j = threadIdx.x - 64;
        scales[a][j] = p.w_scale[min(t.col0 + j, p.n - 1)];
        scales[a][j + 128] = p.w_scale[min(t.col0 + j + 128, p.n - 1)];
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      const bool there = row < p.m;
      const float xs = I8 && there ? p.x_scale[row] : 1.f;
      const int token = there ? p.tokens[row] : -1;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(done0 + 8 * a, (i >> 1) & 1, ERR_GEMM_TMEM_FULL_WAIT));
      if (!ok) continue;
      tc_fence_after();
      if (!p.ranges) s = LogStat{-INFINITY, 0.f, 0.f};
#pragma unroll 1
      for (int c = 0; c < BN && row0 < p.m; c += kChunk) {
        const int n0 = t.col0 + c;
        if (n0 >= t.end) break;
        uint32_t v[32];
        B2_TMEM_LD_32(tmem + a * BN + c + ((uint32_t)(quarter * 32) << 16), v);
        tmem_ld_wait();
        float z[32], largest = -INFINITY;
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = I8 ? (float)(int)v[j] * xs * scales[a][c + j] : __uint_as_float(v[j]);
        if (n0 + 32 > t.end) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (n0 + j >= t.end) z[j] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) largest = fmaxf(largest, z[j]);
        add_terms(s, z, largest);
        if (token >= n0 && token < min(n0 + 32, t.end)) {
          float mine = z[0];
#pragma unroll
          for (int j = 1; j < 32; ++j) mine = token == n0 + j ? z[j] : mine;
          p.token_z[row] = mine;
        }
        if (ALT) {
          // Through shared memory (a row's 128 bytes in the order of the 128-byte swizzle) and out as one copy, which leaves out rows that are not
          // there: stored by the threads, 16 bytes of 32 rows at a time, the logits took 1024 int8 rows x 151936 x 5120 from 626 to 903 us.
          if (there) p.largest[(long long)row * p.ldc + n0 / kChunk] = largest;
          if (lane == 0) tma_store_wait_read0();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(out + lane * 128 + ((j ^ (lane & 7)) << 4)), "f"(z[4 * j]), "f"(z[4 * j + 1]),
                         "f"(z[4 * j + 2]), "f"(z[4 * j + 3])
                         : "memory");
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_z, out, n0, row0);
            tma_store_commit();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(map_rank0(read0 + 8 * a));
        else mbar_arrive(read0 + 8 * a);
      }
      if (there && (!p.ranges || t.col0 + BN >= t.end)) p.part[(long long)t.part * p.m + row] = make_float4(s.m, s.s, s.t, 0.f);
    }
    if (ALT && lane == 0) tma_store_wait0();
  }

  // every thread arrives here on every path
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ a row's tiles together
// (Here and below: no __restrict__ on what the kernel before wrote.  These kernels are launched while it still runs, and a read-only load is for
// memory that nothing writes from a kernel's launch on.)  A CTA takes eight rows: a warp reads four parts of all of them at a time (whole lines), then the lanes' and the warps' results are joined,
// always in the same order.
constexpr int kJoinRows = 8, kJoinWarps = 16;
__global__ void __launch_bounds__(32 * kJoinWarps) score_join_kernel(const float4* part, int parts, const float* token_z,
                                                                     const int* tokens, int m, int n, float* logprob,
                                                                     float* entropy) {
  __shared__ LogStat sh[kJoinWarps][kJoinRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * kJoinRows + lane % kJoinRows;
  pdl_wait();
  LogStat s{-INFINITY, 0.f, 0.f};
  if (row < m)
#pragma unroll 4
    for (int t = warp * 4 + lane / kJoinRows; t < parts; t += 4 * kJoinWarps) {
      const float4 q = part[(long long)t * m + row];
      s = join(s, LogStat{q.x, q.y, q.z});
    }
#pragma unroll
  for (int o = 16; o >= kJoinRows; o >>= 1)
    s = join(s, LogStat{__shfl_down_sync(0xffffffffu, s.m, o), __shfl_down_sync(0xffffffffu, s.s, o), __shfl_down_sync(0xffffffffu, s.t, o)});
  if (lane < kJoinRows) sh[warp][lane] = s;
  __syncthreads();
  if (threadIdx.x < kJoinRows && row < m) {
    LogStat all = sh[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) all = join(all, sh[w][threadIdx.x]);
    const LogNorm norm = log_norm(all);
    const int t = tokens[row];
    logprob[row] = t >= 0 && t < n ? log_prob(norm, token_z[row]) : NAN;
    entropy[row] = norm.entropy;
  }
}

// A CTA takes a row: its parts joined, and the alternatives from the maxima of its chunks and the few chunks that matter.
constexpr int kAltThreads = 256, kAltWarps = kAltThreads / 32, kAltChunks = 1024;
__global__ void __launch_bounds__(kAltThreads) score_alternatives_kernel(const float4* part, int parts, const float* token_z,
                                                                         const int* tokens, int m, int n, const float* z, long long ldz,
                                                                         const float* largest, int ldc, int top, float* logprob,
                                                                         float* entropy, int* top_ids, float* top_logprobs) {
  __shared__ LogStat stat[kAltWarps];
  __shared__ float best_of[kAltWarps][32];
  __shared__ unsigned long long lists[kAltWarps][32];
  __shared__ int count, chosen[kAltChunks];
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, chunks = (n + kChunk - 1) / kChunk;
  pdl_wait();
  z += row * ldz;
  largest += (long long)row * ldc;
  float best = -INFINITY;
#pragma unroll 8
  for (int i = threadIdx.x; i < chunks; i += kAltThreads) best = fmaxf(best, largest[i]);
  LogStat s{-INFINITY, 0.f, 0.f};
#pragma unroll 4
  for (int t = threadIdx.x; t < parts; t += kAltThreads) {
    const float4 q = part[(long long)t * m + row];
    s = join(s, LogStat{q.x, q.y, q.z});
  }
  const float mine = best;
  best = sort_lanes(best, lane);
  best_of[warp][lane] = best;
  s = join_lanes<32>(s);
  if (lane == 0) stat[warp] = s;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
#pragma unroll
  for (int half = kAltWarps / 2; half > 0; half >>= 1) {
    if (warp < half) best_of[warp][lane] = best = merge_floats(best, best_of[warp + half][lane], lane);
    __syncthreads();
  }
  // the top-th largest of the threads' maxima: as many logits reach it
  const float bound = best_of[0][top - 1];
  if (mine >= bound && mine > -INFINITY)
#pragma unroll 8
    for (int i = threadIdx.x; i < chunks; i += kAltThreads) {
      const float x = largest[i];
      if (x >= bound && x > -INFINITY) {
        const int at = atomicAdd(&count, 1);      // (whatever their order, the same logits come out)
        if (at < kAltChunks) chosen[at] = i;
      }
    }
  __syncthreads();
  unsigned long long list = 0, last = 0;
  const bool listed = count <= kAltChunks;      // else (rows of ties) all chunks are looked at again
  constexpr int kAhead = 4;
  const int all = listed ? count : chunks;
  for (int c0 = warp; c0 < all; c0 += kAhead * kAltWarps) {
    float x[kAhead];
    int id[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int c = c0 + j * kAltWarps;
      id[j] = c < all ? (listed ? chosen[c] : c) * kChunk + lane : n;
      x[j] = id[j] < n ? z[id[j]] : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) offer(list, last, x[j] >= bound && x[j] > -INFINITY ? logit_key(x[j], id[j]) : 0, top, lane);
  }
  lists[warp][lane] = list;
  __syncthreads();
#pragma unroll
  for (int half = kAltWarps / 2; half > 0; half >>= 1) {
    if (warp < half) lists[warp][lane] = list = merge_lists(list, lists[warp + half][lane], lane);
    __syncthreads();
  }
  if (warp) return;
  list = fill_list(list, z, n, top, lane);
  const LogNorm norm = log_norm(join_lanes<kAltWarps>(stat[lane % kAltWarps]));
  if (lane == 0) {
    const int t = tokens[row];
    logprob[row] = t >= 0 && t < n ? log_prob(norm, token_z[row]) : NAN;
    entropy[row] = norm.entropy;
  }
  if (lane < top) {
    top_ids[(long long)row * top + lane] = list ? (int)key_id(list) : -1;
    top_logprobs[(long long)row * top + lane] = list ? log_prob(norm, order_value((uint32_t)(list >> 32))) : -INFINITY;
  }
}

// ------------------------------------------------------------------ rows as int8 with a scale per row
// s = max|x| / 127, q = rint(x (1 / s)): 8 bits a value, off by at most s / 2.  A row with a NaN or an infinity has the scale NaN, and so
// have its logits; no scale is below 2^-126, whose inverse is finite.  One CTA per row, 16 bytes a thread and step.
__global__ void __launch_bounds__(256) quant_kernel(const __nv_bfloat16* x, long long ldx, int k, int8_t* q, long long ldq,
                                                    float* scale) {
  __shared__ float part[8];
  pdl_wait();
  const uint4* row = reinterpret_cast<const uint4*>(x + blockIdx.x * ldx);
  const int vecs = k / 8, tail = k % 8;
  const __nv_bfloat16* end = x + blockIdx.x * ldx + vecs * 8;
  float largest = 0.f;
  for (int i = threadIdx.x; i < vecs; i += 256) {
    const uint4 v = row[i];
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
    const uint4 v = row[i];
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

// box_rows rows x 128 bytes of a matrix [rows][cols] of elements of 1 (int8), 2 (bf16) or 4 (fp32) bytes, rows ld elements apart; what lies outside
// reads as zeros and is not written
int make_map(CUtensorMap* map, const void* ptr, int size, int rows, long long cols, long long ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return -100;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * size};
  const cuuint32_t box[2] = {(cuuint32_t)(kStageRow / size), (cuuint32_t)box_rows}, step[2] = {1, 1};
  const CUresult r = fn(map, size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : size == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(ptr), dims, strides, box, step,
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

// How a product is laid out: CTAs by themselves or pairs, ranges of columns or tiles in turn, parts of a row.
struct Layout {
  bool pair;
  int ranges, parts, clusters;
};
int layout_of(int m, int n, Layout& l) {
  if (m < 1 || n < 1 || n > 0x7fff0000) return -1;
  l.pair = m > 3 * BM || (m > BM && m <= 2 * BM);
  const int tiles_m = (m - 1) / (l.pair ? 2 * BM : BM) + 1, tiles_n = (n + BN - 1) / BN, at_once = l.pair ? sm_count() / 2 : sm_count();
  l.ranges = m <= kRangeRows ? min(max(1, at_once / tiles_m), (n + kGrain - 1) / kGrain) : 0;
  l.parts = l.ranges ? l.ranges : tiles_n;
  if ((long long)tiles_m * l.parts > 0x3fffffff) return -1;
  l.clusters = l.ranges ? tiles_m * l.ranges : min(tiles_m * tiles_n, at_once);
  return 0;
}

template <bool I8, bool ALT, bool PAIR>
int launch(const CUtensorMap& mx, const CUtensorMap& me, const CUtensorMap& mw, const CUtensorMap& mg, const CUtensorMap& mz, const ScoreParams& p, int clusters, cudaStream_t st) {
  constexpr int kSmem = Form<PAIR>::SMEM + (ALT ? kOutBytes : 0);
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(score_kernel<I8, ALT, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return (int)e;
    configured[dev & 63] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(PAIR ? 2 * clusters : clusters);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (PAIR) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = 2;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (!b2_no_pdl()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return (int)cudaLaunchKernelEx(&cfg, score_kernel<I8, ALT, PAIR>, mx, me, mw, mg, mz, p);
}
template <bool I8, bool ALT>
int launch(const CUtensorMap& mx, const CUtensorMap& me, const CUtensorMap& mw, const CUtensorMap& mg, const CUtensorMap& mz, const ScoreParams& p, const Layout& l, cudaStream_t st) {
  return l.pair ? launch<I8, ALT, true>(mx, me, mw, mg, mz, p, l.clusters, st) : launch<I8, ALT, false>(mx, me, mw, mg, mz, p, l.clusters, st);
}

// The workspace of a call, in floats from its beginning: sums, tokens' logits; alternatives: logits and their maxima; int8: rows and scales.
struct Room {
  long long token_z, z, largest, scale, q, all;
  int chunks, ldq;
};
Room room_of(const Layout& l, int m, int n, int k, int top, bool i8) {
  const auto lines = [](long long floats) { return (floats + 31) / 32 * 32; };
  Room r;
  r.chunks = (n + kChunk - 1) / kChunk;
  r.ldq = (k + 15) / 16 * 16;
  r.token_z = 4ll * l.parts * m;
  r.z = lines(r.token_z + m);
  r.largest = r.z + (top ? (long long)r.chunks * kChunk * m : 0);
  r.scale = lines(r.largest + (top ? (long long)r.chunks * m : 0));
  r.q = lines(r.scale + (i8 ? m : 0));
  r.all = r.q + (i8 ? (long long)r.ldq / 4 * m : 0);
  return r;
}
}  // namespace

// Floats of workspace for m rows of k against n columns (-1: sizes that are refused): `work`, of one call at a time, 16-byte aligned.
extern "C" long long b2_score_work(int m, int n, int k, int top, int i8) {
  Layout l;
  return layout_of(m, n, l) || k < 1 || k > (i8 ? kMostI8 : 0x7fffff00) ? -1 : room_of(l, m, n, k, top, i8 != 0).all;
}
// Log probabilities of the tokens of bf16 rows x [m][k] against the head w [n][k], entropies and alternatives.  The head is bf16, or int8 (w_scale: of its
// rows), for which the rows are quantised too.  Rows are ldx and ldw elements apart, multiples of 16 bytes, and those of the head of 128 bytes at least.
extern "C" int b2_score(const void* x, long long ldx, const void* w, long long ldw, const float* w_scale, int m, int n, int k, const int* tokens, int top,
                        float* work, float* logprob, float* entropy, int* top_ids, float* top_logprobs, void* stream) {
  const bool i8 = w_scale != nullptr;
  const int size = i8 ? 1 : 2;
  Layout l;
  if (layout_of(m, n, l) || (long long)k * size < kStageRow || k > (i8 ? kMostI8 : 0x7fffff00) || ldx < k || ldw < k || top < 0 || top > kMaxTop) return -1;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)work | (unsigned long long)(ldx * 2) | (unsigned long long)(ldw * size)) & 15) return -3;
  const Room r = room_of(l, m, n, k, top, i8);
  cudaStream_t st = (cudaStream_t)stream;
  ScoreParams p{};
  p.m = m; p.n = n; p.kb = (int)(((long long)k * size + kStageRow - 1) / kStageRow);
  p.ranges = l.ranges;
  p.x_scale = work + r.scale; p.w_scale = w_scale; p.tokens = tokens;
  p.part = (float4*)work; p.token_z = work + r.token_z;
  p.largest = work + r.largest; p.ldc = r.chunks;
  void* q = work + r.q;
  // (a map is a microsecond of the host's: none is made that no block of x, or no tile in ranges that are narrower than one, would use)
  CUtensorMap mx, me, mw, mg, mz;
  const auto map_of_x = [&](CUtensorMap* to, int box) { return i8 ? make_map(to, q, 1, m, k, r.ldq, box) : make_map(to, x, 2, m, k, ldx, box); };
  int rc = m >= BM ? map_of_x(&mx, BM) : 0;
  if (!rc && m % BM) rc = map_of_x(&me, (m % BM + 7) / 8 * 8);
  if (m < BM) mx = me;
  if (m % BM == 0) me = mx;
  const bool narrow = l.ranges && ((n + kGrain - 1) / kGrain + l.ranges - 1) / l.ranges < BN / kGrain;
  if (!rc && !narrow) rc = make_map(&mw, w, size, n, k, ldw, l.pair ? BN / 2 : BN);
  if (!rc && l.ranges) rc = make_map(&mg, w, size, n, k, ldw, l.pair ? kGrain / 2 : kGrain);
  if (narrow) mw = mg;
  if (!l.ranges) mg = mw;
  mz = mw;
  const long long ldz = (long long)r.chunks * kChunk;
  if (!rc && top) rc = make_map(&mz, work + r.z, 4, m, ldz, ldz, 32);
  if (rc) return rc;
  if (i8) {
    rc = b2_launch(quant_kernel, dim3(m), dim3(256), 0, st, true, (const __nv_bfloat16*)x, ldx, k, (int8_t*)q, (long long)r.ldq, work + r.scale);
    if (rc) return rc;
  }
  if (top) rc = i8 ? launch<true, true>(mx, me, mw, mg, mz, p, l, st) : launch<false, true>(mx, me, mw, mg, mz, p, l, st);
  else rc = i8 ? launch<true, false>(mx, me, mw, mg, mz, p, l, st) : launch<false, false>(mx, me, mw, mg, mz, p, l, st);
  if (rc) return rc;
  if (top)
    return b2_launch(score_alternatives_kernel, dim3(m), dim3(kAltThreads), 0, st, true, p.part, l.parts, p.token_z, tokens, m, n, work + r.z, ldz, p.largest, p.ldc,
                     top, logprob, entropy, top_ids, top_logprobs);
  return b2_launch(score_join_kernel, dim3((m + kJoinRows - 1) / kJoinRows), dim3(32 * kJoinWarps), 0, st, true, p.part, l.parts, p.token_z, tokens, m, n,
                   logprob, entropy);
}

B2_DEFINE_STATUS(score)
