// Attention of token trees over a paged cache on tcgen05 / TMEM: row i, a node of its request's tree, sees the request's cached positions
// and its own ancestors (bit j of its mask: node j), whose keys and values stand in the tree's pages.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j      j: cached positions < length, nodes of the mask; with a window those less than
//                                                   `window` positions before the row
//
// A row that sees nothing is 0.  All nodes of a tree share their request's keys, so a key head's queries are one matrix of nodes x (query heads
// per key head) rows, M = 128 of them to a tensor-core tile, and the cache is read once for all: the bytes of K and V are the bound as long as
// the tiles keep up, which they do up to 256 rows (below).
//
// Work.  The cache is cut into tiles of 64 keys; the tree is one more tile behind a request's last.  All tiles of all requests and key heads, one
// after another, are one line, and every CTA takes an equal part of it, whatever the requests' lengths are (they are on the device only).  A part
// begins and ends inside a request as a rule: what it has of one is a segment.  A segment that is all of a request's key head writes results;
// the others leave unnormalised sums against their running maximum, and a second kernel adds them up in the order of the keys.
//
// A CTA: one warp copies (tiled TMA, 16 keys x 64 dims a box, 128-byte swizzle; pages behind the end are asked for outside the tensor and
// come as zeros), one thread per query tile issues the products, a thread per query row does the softmax: scores come from tensor memory, P goes
// back there as the A operand of P V; the accumulator is rescaled only where a row's maximum grew by more than 2^6.  Score buffers are
// double, so that the next scores are under way while a tile's softmax runs.  Up to 128 query rows (NW 1) two CTAs share an SM; beyond (NW 2)
// a CTA has two query tiles that share every K / V tile.  More than 256 rows take further CTAs (blockIdx.y) over the same keys.
// An 8-bit cache comes in as bytes (bulk copies, scales with them), four warps make integers in bf16 of them, which are exact; K's scale goes on
// the scores and V's on the weights, both in fp32.
#include "common.cuh"

using namespace b2;

namespace {

constexpr int kPage = 16, kMaxNodes = 64, kMaxReq = 1024;
constexpr int BQ = 128, BK = 64;

struct TreeAttnParams {
  const __nv_bfloat16* q;
  long long ldq;
  const int8_t *k8, *v8;           // 8-bit form
  const float *k_scale, *v_scale;
  const int *lengths, *row_start, *row_req, *row_pos, *block_table, *tree_table;
  const unsigned long long* masks;
  int B, max_blocks, tree_blocks, num_pages, rows, n_q, n_kv, gqa, window;
  int group_tokens;                // nodes to a CTA's query tiles
  float scale_log2;
  __nv_bfloat16* out;
  long long ldo;
  float *part_o, *part_ml;         // [group][column][2][NW x 128 rows][D], and maximum and sum
  int* sched;                      // tiles a column, then the requests' first tiles (of one key head)
};

template <int NDK_, bool I8_, int NW_>
struct Form {
  static constexpr int NDK = NDK_, NW = NW_, D = NDK_ * 64;
  static constexpr bool I8 = I8_;
  static constexpr int T_BYTES = BK * NDK * 128;                 // a K or V tile: [64-dim blocks][64 keys][128 bytes]
  static constexpr int KVS = I8_ ? NW_ : (NW_ == 1 ? (NDK_ == 1 ? 4 : 2) : 4);      // operand tiles
  static constexpr int RS = I8_ ? (NW_ == 1 ? (NDK_ == 1 ? 4 : 2) : 4) : 0;         // stages of bytes
  static constexpr int S_BYTES = 2 * BK * D + 2 * BK * 4;        // keys, values, their scales
  static constexpr int Q_BYTES = NW * BQ * NDK * 128;
  static constexpr int kMma = 1, kSoft = 1 + NW, kConv = kSoft + 4 * NW, kWarps = kConv + (I8_ ? 4 : 0), kThreads = kWarps * 32;
  static constexpr int TMEM = NW == 1 ? 256 : 512;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + KVS * T_BYTES, OFF_ST = OFF_V + KVS * T_BYTES, OFF_SC = OFF_ST + RS * S_BYTES,
                       OFF_CUM = OFF_SC + (I8_ ? 4 * 2 * BK * 4 : 0), OFF_BAR = OFF_CUM + (kMaxReq + 8) * 4, SMEM = OFF_BAR + 512 + 1024;
  static_assert(SMEM <= (NW == 1 ? 115712 : 227 * 1024), "shared memory");
};

// V as an MN-major operand: rows are keys of 128 bytes (64 dims), 8-key groups 1024 bytes apart, the next 64 dims a block further.
__device__ __forceinline__ uint64_t make_desc_v(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
  d |= (uint64_t)((BK * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ void st_32(uint32_t taddr, const uint32_t (&r)[32]) { B2_TMEM_ST_32(taddr, r); }

__device__ __forceinline__ uint32_t bytes_bf16(uint32_t w) {      // even bytes as integers in bf16: 128 + (b & 127) less 128, or 256 where the sign is set
  uint32_t lo = (w & 0x007f007fu) | 0x43004300u, hi = (w & 0x00800080u) | 0x43004300u, d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(lo), "r"(hi));
  return d;
}

// A request as the roles see it.
struct Req {
  int b, r0, n, length, first, nt;      // first row, nodes, cached positions, first tile of the cache that is read, tiles (the tree's is the last)
};

__device__ __forceinline__ int first_tile(const TreeAttnParams& p, int length) { return p.window > 0 ? max(0, length - p.window + 1) / BK : 0; }
__device__ __forceinline__ int nodes_of(const TreeAttnParams& p, int b, int& r0) {
  r0 = p.row_start[b];
  return max(0, min(min(p.row_start[b + 1], p.rows) - r0, kMaxNodes));
}

// The segments of a CTA's part [u, u1) of the line of tiles.
struct Walk {
  long long u, u0, u1;
  int b;
  Req r;
  int h, ts, count, tok;       // key head, first tile and tiles of the segment, nodes of the CTA's group
};

template <class F>
__device__ __forceinline__ bool next_segment(const TreeAttnParams& p, const int* s_cum, Walk& k) {
  for (;;) {
    if (k.u >= k.u1) return false;
    while ((long long)s_cum[k.b + 1] * p.n_kv <= k.u) ++k.b;
    const int nt = s_cum[k.b + 1] - s_cum[k.b];
    const long long rel = k.u - (long long)s_cum[k.b] * p.n_kv;
    k.h = (int)(rel / nt);
    k.ts = (int)(rel - (long long)k.h * nt);
    k.count = (int)min((long long)(nt - k.ts), k.u1 - k.u);
    k.u += k.count;
    k.r.b = k.b;
    k.r.n = nodes_of(p, k.b, k.r.r0);
    k.r.length = p.lengths[k.b];
    k.r.first = first_tile(p, k.r.length);
    k.r.nt = nt;
    k.tok = min(p.group_tokens, k.r.n - (int)blockIdx.y * p.group_tokens);
    if (k.tok > 0) return true;
  }
}

template <class F>
__global__ void __launch_bounds__(F::kThreads, F::NW == 1 ? 2 : 1)
tree_attn_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TreeAttnParams p) {
  constexpr int NDK = F::NDK, NW = F::NW, KVS = F::KVS, D = F::D, RS = F::I8 ? F::RS : 1;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_s = base, k_s0 = base + F::OFF_K, v_s0 = base + F::OFF_V, st_s0 = base + F::OFF_ST, bars = base + F::OFF_BAR;
  int* const s_cum = reinterpret_cast<int*>(gen + F::OFF_CUM);
  float* const s_scale = reinterpret_cast<float*>(gen + F::OFF_SC);       // [4][K, V][64]
  const uint32_t b_kfull = bars, b_kempty = bars + 32, b_vfull = bars + 64, b_vempty = bars + 96, b_rfull = bars + 128, b_rempty = bars + 160;
  auto b_q = [&](int w) { return bars + 192 + w * 8; };
  auto b_sfull = [&](int w, int s) { return bars + 208 + (w * 2 + s) * 8; };
  auto b_pfull = [&](int w, int s) { return bars + 240 + (w * 2 + s) * 8; };
  auto b_odone = [&](int w, int s) { return bars + 272 + (w * 2 + s) * 8; };
  auto b_scale = [&](int g) { return bars + 304 + (g & 3) * 8; };
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(gen + F::OFF_BAR + 344);
  int* const s_sums = reinterpret_cast<int*>(gen + F::OFF_BAR + 384);      // [16]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < KVS; ++i) {
      mbar_init(b_kfull + 8 * i, F::I8 ? 128 : 1);
      mbar_init(b_kempty + 8 * i, NW);
      mbar_init(b_vfull + 8 * i, F::I8 ? 128 : 1);
      mbar_init(b_vempty + 8 * i, NW);
    }
    if (F::I8) {
      for (int i = 0; i < RS; ++i) {
        mbar_init(b_rfull + 8 * i, 1);
        mbar_init(b_rempty + 8 * i, 128);
      }
      for (int i = 0; i < 4; ++i) mbar_init(b_scale(i), 128);
    }
    for (int w = 0; w < NW; ++w) {
      mbar_init(b_q(w), 128);
      for (int s = 0; s < 2; ++s) {
        mbar_init(b_sfull(w, s), 1);
        mbar_init(b_pfull(w, s), 128);
        mbar_init(b_odone(w, s), 1);
      }
    }
    mbar_fence_init();
    if (!F::I8) {
      prefetch_tmap(&map_k);
      prefetch_tmap(&map_v);
    }
  }
  if (warp == F::kMma) {
    tmem_alloc(smem_u32(tmem_slot), F::TMEM);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch_dependents();
  // ---- tiles of one key head before every request
  {
    const int per = (p.B + F::kThreads - 1) / F::kThreads, b0 = tid * per;
    int mine = 0;
    for (int b = b0; b < min(b0 + per, p.B); ++b) {
      int r0;
      const int length = p.lengths[b], n = nodes_of(p, b, r0);
      const int nt = n > 0 ? (length + BK - 1) / BK - first_tile(p, length) + 1 : 0;
      s_cum[b + 1] = mine += nt;
    }
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_sums[warp] = x;
    __syncthreads();
    int before = x - mine;
    for (int w = 0; w < warp; ++w) before += s_sums[w];
    for (int b = b0; b < min(b0 + per, p.B); ++b) s_cum[b + 1] += before;
    if (tid == 0) s_cum[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  auto t_s = [&](int w, int s) { return tmem_base + (uint32_t)(w * 2 + s) * BK; };
  auto t_o = [&](int w) { return tmem_base + (uint32_t)(NW * 2 * BK + w * D); };

  const long long total = (long long)s_cum[p.B] * p.n_kv, each = (total + gridDim.x - 1) / gridDim.x;
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    for (int b = tid; b <= p.B; b += F::kThreads) p.sched[b + 1] = s_cum[b];
    if (tid == 0) p.sched[0] = (int)each;
  }
  Walk k;
  k.u0 = k.u = min(total, blockIdx.x * each);
  k.u1 = min(total, k.u0 + each);
  {
    int lo = 0, hi = p.B - 1;      // the last request that begins at or before u0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)s_cum[mid] * p.n_kv <= k.u0) lo = mid; else hi = mid - 1;
    }
    k.b = lo;
  }

  if (warp == 0) {
    // ---------------------------------------------------------- copies: lanes issue one box (bf16) or one run of bytes (8-bit) each
    bool ok = true;
    int g = 0;
    while (ok && next_segment<F>(p, s_cum, k)) {
      const int limit = min((k.r.length + kPage - 1) / kPage, p.max_blocks), tree_pages = (k.r.n + kPage - 1) / kPage;
      const int* bt = p.block_table + (size_t)k.r.b * p.max_blocks;
      auto entry = [&](int i) {      // (what names no page reads as page 0, which is nobody's; behind the end there is none)
        const int page = i < limit ? bt[i] : -1;
        return i < limit && (page < 0 || page >= p.num_pages) ? 0 : page;
      };
      int at = ((k.r.first + k.ts) * 4) & ~31;             // pages at .. at + 31 are in the lanes
      int ids = entry(at + lane), ahead = entry(at + 32 + lane);
      int tree_ids = lane < min(tree_pages, p.tree_blocks) ? p.tree_table[(size_t)k.r.b * p.tree_blocks + lane] : -1;
      if (lane < tree_pages && (tree_ids < 0 || tree_ids >= p.num_pages)) tree_ids = 0;
      for (int i = 0; i < k.count; ++i, ++g) {
        const int t = k.ts + i;
        const bool tree = t == k.r.nt - 1;
        const int pi = (k.r.first + t) * 4;
        if (!tree && pi >= at + 32) {
          at += 32;
          ids = ahead;
          ahead = entry(at + 32 + lane);
        }
        const int pg = F::I8 ? (lane >> 2) & 3 : (lane / NDK) & 3;
        int page = __shfl_sync(0xffffffffu, tree ? tree_ids : ids, tree ? pg : pi - at + pg);
        const bool there = page >= 0;
        if constexpr (F::I8) {
          const int s = g % RS;
          const uint32_t full = b_rfull + 8 * s, st = st_s0 + s * F::S_BYTES;
          if (g >= RS) ok = mbar_wait(b_rempty + 8 * s, ((g / RS) & 1) ^ 1, ERR_ATTN_WAIT);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          const int pages = __popc(__ballot_sync(0xffffffffu, lane < 16 && there)) >> 2;
          if (lane == 0) mbar_expect_tx(full, pages * (2 * kPage * D + 2 * kPage * 4));
          __syncwarp();
          if (lane < 16 && there) {
            const long long row = ((long long)page * p.n_kv + k.h) * kPage;
            const int which = lane & 3;
            if (which < 2) bulk_g2s(st + which * (BK * D) + pg * (kPage * D), (which ? p.v8 : p.k8) + row * D, kPage * D, full);
            else bulk_g2s(st + 2 * BK * D + (which - 2) * (BK * 4) + pg * (kPage * 4), (which == 3 ? p.v_scale : p.k_scale) + row, kPage * 4, full);
          }
        } else {
          const int s = g % KVS, ph = (g / KVS) & 1;
          const int row = there ? (page * p.n_kv + k.h) * kPage : p.num_pages * p.n_kv * kPage, c = lane % NDK;
          const uint32_t dst = s * F::T_BYTES + c * (BK * 128) + pg * (kPage * 128);
          if (g >= KVS) ok = mbar_wait(b_kempty + 8 * s, ph ^ 1, ERR_ATTN_WAIT);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          if (lane == 0) mbar_expect_tx(b_kfull + 8 * s, F::T_BYTES);
          __syncwarp();
          if (lane < 4 * NDK) tma_load_2d(k_s0 + dst, &map_k, c * 64, row, b_kfull + 8 * s);
          if (g >= KVS) ok = mbar_wait(b_vempty + 8 * s, ph ^ 1, ERR_ATTN_WAIT);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            mbar_wait(b_kfull + 8 * s, ph, ERR_ATTN_WAIT);      // the K copies just issued
            break;
          }
          if (lane == 0) mbar_expect_tx(b_vfull + 8 * s, F::T_BYTES);
          __syncwarp();
          if (lane < 4 * NDK) tma_load_2d(v_s0 + dst, &map_v, c * 64, row, b_vfull + 8 * s);
        }
      }
    }
    if (!ok) {      // copies in flight end before the CTA does
      if constexpr (F::I8)
        for (int i = max(0, g - RS); i < g; ++i) mbar_wait(b_rfull + 8 * (i % RS), (i / RS) & 1, ERR_ATTN_WAIT);
      else
        for (int i = max(0, g - KVS); i < g; ++i) {
          mbar_wait(b_kfull + 8 * (i % KVS), (i / KVS) & 1, ERR_ATTN_WAIT);
          mbar_wait(b_vfull + 8 * (i % KVS), (i / KVS) & 1, ERR_ATTN_WAIT);
        }
    }
  } else if (warp < F::kSoft) {
    // ---------------------------------------------------------- products of query tile w
    const int w = warp - F::kMma;
    constexpr uint32_t idesc_qk = make_idesc(1, 1, BQ, BK);
    constexpr uint32_t idesc_pv = make_idesc(1, 1, BQ, D) | (1u << 16);      // V is MN-major
    const uint32_t hi_k = (uint32_t)(make_desc_sw128(0) >> 32), hi_v = (uint32_t)(make_desc_v(0) >> 32);
    const uint32_t ql = (uint32_t)make_desc_sw128(q_s + w * (BQ * NDK * 128)), k_lo = (uint32_t)make_desc_sw128(k_s0), v_lo = (uint32_t)make_desc_v(v_s0);
    auto issue_qk = [&](int j) -> bool {
      const int s = j & 1, ks = j % KVS;
      if (!mbar_wait(b_kfull + 8 * ks, (j / KVS) & 1, ERR_ATTN_WAIT)) return false;
      if (j >= 2 && !mbar_wait(b_odone(w, s), ((j >> 1) - 1) & 1, ERR_ATTN_WAIT)) return false;      // the buffer holds P(j - 2) until its product has read it
      tc_fence_after();
      const uint32_t kl = k_lo + ks * (F::T_BYTES >> 4), ts = t_s(w, s);
#pragma unroll
      for (int x = 0; x < 4 * NDK; ++x)
        umma_f16_w(ts, ql + (((x >> 2) * (BQ * 128) + (x & 3) * 32) >> 4), hi_k, kl + (((x >> 2) * (BK * 128) + (x & 3) * 32) >> 4), hi_k, idesc_qk, x != 0);
      tc_commit(b_sfull(w, s));
      tc_commit(b_kempty + 8 * ks);
      return true;
    };
    bool ok = true;
    int g = 0, seg = 0;
    while (ok && next_segment<F>(p, s_cum, k)) {
      if (lane == 0) {
        ok = mbar_wait(b_q(w), seg & 1, ERR_ATTN_WAIT);
        if (ok) ok = issue_qk(g);
      }
      for (int i = 0; i < k.count; ++i, ++g) {
        const int s = g & 1, ks = g % KVS, t = k.ts + i;
        const int valid = t == k.r.nt - 1 ? k.r.n : min(BK, k.r.length - (k.r.first + t) * BK);
        const bool tail = !F::I8 && (valid & 15) != 0;
        if (lane == 0) {
          if (ok && i + 1 < k.count) ok = issue_qk(g + 1);
          if (ok) ok = mbar_wait(b_pfull(w, s), (g >> 1) & 1, ERR_ATTN_WAIT);
          if (ok) ok = mbar_wait(b_vfull + 8 * ks, (g / KVS) & 1, ERR_ATTN_WAIT);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        if (tail) {
          // values behind the last key's are anything: their weights are 0, but 0 x infinity is not
          if (!mbar_wait(b_vfull + 8 * ks, (g / KVS) & 1, ERR_ATTN_WAIT)) ok = false;      // (over: every lane sees the copies)
          const int end = (valid + 15) & ~15;
          for (int x = lane; x < (end - valid) * NDK * 8; x += 32) {
            const int row = valid + x / (NDK * 8), c = x % (NDK * 8);
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(v_s0 + ks * F::T_BYTES + (c >> 3) * (BK * 128) + row * 128 + (c & 7) * 16), "r"(0) : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          tc_fence_after();
          const uint32_t vl = v_lo + ks * (F::T_BYTES >> 4), tp = t_s(w, s);
#pragma unroll
          for (int x = 0; x < 4; ++x)      // 16 keys a step; P in tensor memory, 8 columns of pairs
            umma_f16_ts_w(t_o(w), tp + 8 * x, vl + ((x * 16 * 128) >> 4), hi_v, idesc_pv, (i | x) != 0);
          tc_commit(b_odone(w, s));
          tc_commit(b_vempty + 8 * ks);
        }
      }
      ++seg;
    }
  } else if (warp < F::kConv) {
    // ---------------------------------------------------------- softmax: a thread per query row of tile w
    constexpr float kLazy = 6.f;
    const int w = (warp - F::kSoft) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    bool ok = true;
    int g = 0;
    while (ok && next_segment<F>(p, s_cum, k)) {
      const int rr = w * BQ + r, live_rows = k.tok * p.gqa;
      const bool row_ok = rr < live_rows, warp_ok = w * BQ + quarter * 32 < live_rows;
      const int node = blockIdx.y * p.group_tokens + rr / p.gqa, head = k.h * p.gqa + rr % p.gqa, row = k.r.r0 + node;
      // ---- the row's query (the products of the segment before have read theirs: their scores were here)
      if (row_ok) {
        const uint4* src = reinterpret_cast<const uint4*>(p.q + row * p.ldq + head * D);
        uint4 x[8 * NDK];
#pragma unroll
        for (int c = 0; c < 8 * NDK; ++c) x[c] = src[c];
#pragma unroll
        for (int c = 0; c < 8 * NDK; ++c)
          *reinterpret_cast<uint4*>(gen + w * (BQ * NDK * 128) + (c >> 3) * (BQ * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x[c];
      }
      fence_proxy_async_smem();
      mbar_arrive(b_q(w));
      const int pos = row_ok && p.window > 0 ? p.row_pos[row] : 0, lo = p.window > 0 ? pos - p.window + 1 : 0;      // the first position that is seen
      unsigned long long mask = 0;
      if (row_ok && k.ts + k.count == k.r.nt) {
        mask = p.masks[row];
        if (k.r.n < 64) mask &= (1ull << k.r.n) - 1;
        if (lo > k.r.length)
          for (int j = 0; j < k.r.n; ++j)
            if (p.row_pos[k.r.r0 + j] < lo) mask &= ~(1ull << j);
      }
      float mref = -INFINITY, l = 0.f;
      for (int i = 0; i < k.count; ++i, ++g) {
        const int s = g & 1, t = k.ts + i;
        if (ok) ok = mbar_wait(b_sfull(w, s), (g >> 1) & 1, ERR_ATTN_WAIT);
        if (!ok) break;
        if (!warp_ok) {      // rows of nobody: the products take what is there
          mbar_arrive(b_pfull(w, s));
          continue;
        }
        if (F::I8) ok = mbar_wait(b_scale(g), (g >> 2) & 1, ERR_ATTN_WAIT);
        tc_fence_after();
        unsigned long long vis = mask;
        if (t != k.r.nt - 1) {
          const int key0 = (k.r.first + t) * BK, end = min(BK, k.r.length - key0), begin = max(0, lo - key0);
          vis = end >= BK ? ~0ull : (1ull << end) - 1;
          if (begin > 0) vis = begin >= BK ? 0ull : vis & (~0ull << begin);
        }
        uint32_t v[2][32];
        B2_TMEM_LD_32(t_s(w, s) + lane_addr, v[0]);
        B2_TMEM_LD_32(t_s(w, s) + lane_addr + 32, v[1]);
        tmem_ld_wait();
        const float* sc = s_scale + (g & 3) * (2 * BK);
        if constexpr (F::I8) {
#pragma unroll
          for (int j = 0; j < 64; j += 4) {
            const float4 f = *reinterpret_cast<const float4*>(sc + j);
            const float ff[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j >> 5][(j & 31) + e] = __float_as_uint(__uint_as_float(v[j >> 5][(j & 31) + e]) * ff[e]);
          }
        }
        if (__any_sync(0xffffffffu, vis != ~0ull)) {
          const uint32_t half[2] = {(uint32_t)vis, (uint32_t)(vis >> 32)};
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (!(half[j >> 5] >> (j & 31) & 1)) v[j >> 5][j & 31] = 0xff800000u;
        }
        float ma = -INFINITY, mb = -INFINITY;
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          asm("max.f32 %0, %0, %1, %2;" : "+f"(ma) : "f"(__uint_as_float(v[0][j])), "f"(__uint_as_float(v[0][j + 1])));
          asm("max.f32 %0, %0, %1, %2;" : "+f"(mb) : "f"(__uint_as_float(v[1][j])), "f"(__uint_as_float(v[1][j + 1])));
        }
        const float factor = F::I8 ? 1.f : p.scale_log2;
        const float tmax = fmaxf(ma, mb) * factor;
        float alpha = 1.f;
        if (tmax > mref + kLazy || (mref == -INFINITY && tmax > -INFINITY)) {
          alpha = exp2f(mref - tmax);      // 0 at the row's first key
          mref = tmax;
        }
        const float nm = mref == -INFINITY ? 0.f : -mref;
        if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          ok = mbar_wait(b_odone(w, s ^ 1), ((g - 1) >> 1) & 1, ERR_ATTN_WAIT);
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 2 * NDK; ++c) {
            uint32_t o[32];
            B2_TMEM_LD_32(t_o(w) + lane_addr + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
            B2_TMEM_ST_32(t_o(w) + lane_addr + c * 32, o);
          }
          tmem_st_wait();
        }
        unsigned long long sc2, nm2, acc0 = 0ull, acc1 = 0ull;
        asm("mov.b64 %0, {%1, %1};" : "=l"(sc2) : "f"(factor));
        asm("mov.b64 %0, {%1, %1};" : "=l"(nm2) : "f"(nm));
        uint32_t pk[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          unsigned long long xy;
          asm("mov.b64 %0, {%1, %2};" : "=l"(xy) : "r"(v[j >> 4][(2 * j) & 31]), "r"(v[j >> 4][(2 * j + 1) & 31]));
          if (F::I8) asm("add.rn.f32x2 %0, %0, %1;" : "+l"(xy) : "l"(nm2));
          else asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(xy) : "l"(sc2), "l"(nm2));
          float x0, x1, e0, e1;
          asm("mov.b64 {%0, %1}, %2;" : "=f"(x0), "=f"(x1) : "l"(xy));
          asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(x0));
          asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(x1));
          unsigned long long ee;
          asm("mov.b64 %0, {%1, %2};" : "=l"(ee) : "f"(e0), "f"(e1));
          if (j & 1) asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc1) : "l"(ee));
          else asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc0) : "l"(ee));
          if constexpr (F::I8) {
            const float2 f = *reinterpret_cast<const float2*>(sc + BK + 2 * j);
            // (a weight of nothing stays nothing, whatever the scale behind the last key is)
            pk[j] = pack_bf16(e0 > 0.f ? e0 * f.x : 0.f, e1 > 0.f ? e1 * f.y : 0.f);
          } else {
            pk[j] = pack_bf16(e0, e1);
          }
        }
        st_32(t_s(w, s) + lane_addr, pk);
        tmem_st_wait();
        float a0, a1, a2, a3;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(acc0));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a2), "=f"(a3) : "l"(acc1));
        l = l * alpha + (a0 + a1) + (a2 + a3);
        tc_fence_before();
        mbar_arrive(b_pfull(w, s));
      }
      if (!ok) break;
      // ---- the segment's sums, once its last product is done
      ok = mbar_wait(b_odone(w, (g - 1) & 1), ((g - 1) >> 1) & 1, ERR_ATTN_WAIT);
      if (!ok) break;
      tc_fence_after();
      if (warp_ok) {
        const bool whole = k.count == k.r.nt;
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const size_t slot = (((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + (k.u - k.count != k.u0)) * (NW * BQ) + rr;
        __nv_bfloat16* dst = p.out + row * p.ldo + head * D;
#pragma unroll 1
        for (int c = 0; c < 2 * NDK; ++c) {
          uint32_t o[32];
          B2_TMEM_LD_32(t_o(w) + lane_addr + c * 32, o);
          tmem_ld_wait();
          if (!row_ok) continue;
          if (whole) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<uint4*>(dst + c * 32 + 8 * j) = make_uint4(
                  pack_bf16(__uint_as_float(o[8 * j]) * inv, __uint_as_float(o[8 * j + 1]) * inv), pack_bf16(__uint_as_float(o[8 * j + 2]) * inv, __uint_as_float(o[8 * j + 3]) * inv),
                  pack_bf16(__uint_as_float(o[8 * j + 4]) * inv, __uint_as_float(o[8 * j + 5]) * inv), pack_bf16(__uint_as_float(o[8 * j + 6]) * inv, __uint_as_float(o[8 * j + 7]) * inv));
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(p.part_o + slot * D + c * 32 + 4 * j) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
        }
        if (!whole && row_ok) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(mref, l);
      }
      tc_fence_before();
    }
  } else if constexpr (F::I8) {
    // ---------------------------------------------------------- bytes to integers in bf16: a thread's piece is 16 bytes of a key
    const int ct = tid - F::kConv * 32;
    bool ok = true;
    int g = 0;
    auto expand = [&](uint32_t src, uint32_t dst) {
#pragma unroll
      for (int x = ct; x < BK * D / 16; x += 128) {
        const int row = x / (D / 16), c = x % (D / 16);
        uint32_t ww[4], o[8];
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(ww[0]), "=r"(ww[1]), "=r"(ww[2]), "=r"(ww[3]) : "r"(src + x * 16));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t ev = bytes_bf16(ww[j]), od = bytes_bf16(ww[j] >> 8);
          o[2 * j] = __byte_perm(ev, od, 0x5410);
          o[2 * j + 1] = __byte_perm(ev, od, 0x7632);
        }
        // (the second 64 dims' pieces go the other way round, so that eight threads' stores meet eight banks of 16 bytes)
        const uint32_t to = dst + (c >> 2) * (BK * 128) + row * 128;
        const int c0 = (2 * c) & 7, turn = (c >> 2) & 1;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int y = e ^ turn;
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to + (((c0 + y) ^ (row & 7)) << 4)), "r"(y ? o[4] : o[0]), "r"(y ? o[5] : o[1]), "r"(y ? o[6] : o[2]),
                       "r"(y ? o[7] : o[3])
                       : "memory");
        }
      }
      fence_proxy_async_smem();
    };
    while (ok && next_segment<F>(p, s_cum, k))
      for (int i = 0; i < k.count; ++i, ++g) {
        const int rs = g % RS, ks = g % KVS, ph = ((g / KVS) & 1) ^ 1;
        const uint32_t st = st_s0 + rs * F::S_BYTES;
        ok = mbar_wait(b_rfull + 8 * rs, (g / RS) & 1, ERR_ATTN_WAIT);
        if (ok && g >= KVS) ok = mbar_wait(b_kempty + 8 * ks, ph, ERR_ATTN_WAIT);
        if (!ok) break;
        // the scales of tile g - 4 are read: the place of its keys came free with the scores of tile g - KVS, which waited for the product of
        // tile g - KVS - 2 at least
        const float f = *reinterpret_cast<const float*>(gen + F::OFF_ST + rs * F::S_BYTES + 2 * BK * D + ct * 4);
        s_scale[(g & 3) * (2 * BK) + ct] = ct < BK ? f * p.scale_log2 : f;
        mbar_arrive(b_scale(g));
        expand(st, k_s0 + ks * F::T_BYTES);
        mbar_arrive(b_kfull + 8 * ks);
        if (g >= KVS) ok = mbar_wait(b_vempty + 8 * ks, ph, ERR_ATTN_WAIT);
        if (!ok) break;
        expand(st + BK * D, v_s0 + ks * F::T_BYTES);
        mbar_arrive(b_vfull + 8 * ks);
        mbar_arrive(b_rempty + 8 * rs);
      }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == F::kMma) {
    tc_fence_after();
    tmem_dealloc(tmem_base, F::TMEM);
  }
}

// Segments of a row's head, added up in the order of the keys: a warp per row and head.
template <int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeAttnParams p, int columns, int slot_rows) {
  constexpr int E = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int item = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int row = item / p.n_q, head = item - row * p.n_q;
  if (row >= p.rows) return;
  const int b = p.row_req[row];
  if (b < 0 || b >= p.B) return;
  const long long each = p.sched[0];
  const int before = p.sched[1 + b], nt = p.sched[2 + b] - before;
  const int h = head / p.gqa, node = row - p.row_start[b], z = node / p.group_tokens, rr = (node - z * p.group_tokens) * p.gqa + head % p.gqa;
  if (nt < 1 || node < 0 || node >= kMaxNodes) return;
  const long long a = (long long)before * p.n_kv + (long long)h * nt, e = a + nt;
  const int c0 = (int)(a / each), c1 = (int)((e - 1) / each);
  if (c0 == c1) return;      // one segment: its CTA wrote the result
  auto slot = [&](int c) { return (((size_t)z * columns + c) * 2 + (a > c * each)) * slot_rows + rr; };
  float best = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) best = fmaxf(best, p.part_ml[slot(c) * 2]);
  best = warp_max(best);
  float sum = 0.f, acc[E] = {};
  for (int c = c0; c <= c1; c += 32) {
    float f = 0.f;
    if (c + lane <= c1) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot(c + lane) * 2);
      f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - best);
      sum += f * ml.y;
    }
    const int n = min(32, c1 - c + 1);
    for (int j = 0; j < n; j += 8) {
      float x[8][E];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const float* src = p.part_o + slot(min(c + j + y, c1)) * D + lane * E;
        if constexpr (E == 4) *reinterpret_cast<float4*>(x[y]) = *reinterpret_cast<const float4*>(src);
        else *reinterpret_cast<float2*>(x[y]) = *reinterpret_cast<const float2*>(src);
      }
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const float fy = __shfl_sync(0xffffffffu, f, (j + y) & 31);
#pragma unroll
        for (int d = 0; d < E; ++d) acc[d] += j + y < n && fy > 0.f ? fy * x[y][d] : 0.f;
      }
    }
  }
  sum = warp_sum(sum);
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  __nv_bfloat16* dst = p.out + row * p.ldo + head * D + lane * E;
  if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
  else *reinterpret_cast<uint32_t*>(dst) = pack_bf16(acc[0] * inv, acc[1] * inv);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres);
    return e == cudaSuccess && qres == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(ptr) : nullptr;
  }();
  return fn;
}
int cache_map(CUtensorMap* map, const void* ptr, uint64_t rows, int d) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return -100;
  const cuuint64_t dims[2] = {(cuuint64_t)d, rows}, strides[1] = {(cuuint64_t)d * 2};
  const cuuint32_t box[2] = {64, kPage}, estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -101;
}

int sm_count() {
  static int count[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  int n = count[dev & 63];
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    count[dev & 63] = n;
  }
  return n;
}

// Query tiles of a CTA, nodes to a CTA, CTAs over the same keys, columns of CTAs.
struct Shape {
  int nw, tokens, groups, columns;
};
Shape shape_of(int B, int max_blocks, int n_kv, int gqa, int max_nodes) {
  Shape s;
  s.nw = max_nodes * gqa <= BQ ? 1 : 2;
  const int most = s.nw * BQ / gqa;
  s.groups = (max_nodes + most - 1) / most;
  s.tokens = (max_nodes + s.groups - 1) / s.groups;
  const long long units = (long long)B * n_kv * (max_blocks / 4 + 2);      // tiles there can be
  const long long c = (long long)sm_count() * (s.nw == 1 ? 2 : 1) / s.groups;
  s.columns = (int)(c < 1 ? 1 : c < units ? c : units);
  return s;
}

template <class F>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const TreeAttnParams& p, const Shape& s, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(tree_attn_kernel<F>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
    if (e != cudaSuccess) return (int)e;
    configured[dev & 63] = true;
  }
  const int rc = b2_launch(tree_attn_kernel<F>, dim3(s.columns, s.groups), dim3(F::kThreads), F::SMEM, st, true, mk, mv, p);
  if (rc) return rc;
  const long long items = (long long)p.rows * p.n_q;
  return b2_launch(tree_merge_kernel<F::D>, dim3((unsigned)((items + 7) / 8)), dim3(256), 0, st, true, p, s.columns, s.nw * BQ);
}

}  // namespace

// fp32 words of workspace for b2_tree_attention
extern "C" long long b2_tree_attention_work(int B, int max_blocks, int n_q, int n_kv, int D, int max_nodes) {
  const Shape s = shape_of(B, max_blocks, n_kv, n_q / n_kv, max_nodes);
  return 2ll * s.groups * s.columns * s.nw * BQ * (D + 2) + (B + 2 + 3) / 4 * 4;
}

extern "C" int b2_tree_attention(const void* q, long long ldq, const void* k, const void* v, const float* k_scale, const float* v_scale, const int* lengths,
                                 const int* row_start, const int* row_req, const int* row_pos, const int* block_table, const int* tree_table,
                                 const void* masks, void* out, float* work, long long ldo, int rows, int B, int max_blocks, int tree_blocks, int num_pages,
                                 int n_q, int n_kv, int D, int max_nodes, int window, float scale, void* stream) {
  if (rows < 1 || B < 1 || B > kMaxReq || n_q < 1 || n_kv < 1 || n_q % n_kv || n_q / n_kv > 64 || (D != 64 && D != 128) || max_nodes < 1 || max_nodes > kMaxNodes || num_pages < 1)
    return -1;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)work | (uintptr_t)k_scale | (uintptr_t)v_scale) % 16 || ldq % 8 || ldo % 8) return -2;
  const Shape s = shape_of(B, max_blocks, n_kv, n_q / n_kv, max_nodes);
  TreeAttnParams p;
  p.q = (const __nv_bfloat16*)q; p.ldq = ldq; p.k8 = (const int8_t*)k; p.v8 = (const int8_t*)v; p.k_scale = k_scale; p.v_scale = v_scale;
  p.lengths = lengths; p.row_start = row_start; p.row_req = row_req; p.row_pos = row_pos; p.block_table = block_table; p.tree_table = tree_table;
  p.masks = (const unsigned long long*)masks; p.B = B; p.max_blocks = max_blocks; p.tree_blocks = tree_blocks; p.num_pages = num_pages; p.rows = rows;
  p.n_q = n_q; p.n_kv = n_kv; p.gqa = n_q / n_kv; p.window = window; p.group_tokens = s.tokens; p.scale_log2 = scale * 1.4426950408889634f;
  p.out = (__nv_bfloat16*)out; p.ldo = ldo;
  const size_t slots = 2ull * s.groups * s.columns * s.nw * BQ;
  p.part_o = work; p.part_ml = work + slots * D; p.sched = reinterpret_cast<int*>(work + slots * (D + 2));
  CUtensorMap mk = {}, mv = {};
  if (!k_scale) {
    int rc = cache_map(&mk, k, (uint64_t)num_pages * n_kv * kPage, D);
    if (!rc) rc = cache_map(&mv, v, (uint64_t)num_pages * n_kv * kPage, D);
    if (rc) return rc;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  switch ((D == 128 ? 4 : 0) + (k_scale ? 2 : 0) + s.nw - 1) {
    case 0: return launch<Form<1, false, 1>>(mk, mv, p, s, st);
    case 1: return launch<Form<1, false, 2>>(mk, mv, p, s, st);
    case 2: return launch<Form<1, true, 1>>(mk, mv, p, s, st);
    case 3: return launch<Form<1, true, 2>>(mk, mv, p, s, st);
    case 4: return launch<Form<2, false, 1>>(mk, mv, p, s, st);
    case 5: return launch<Form<2, false, 2>>(mk, mv, p, s, st);
    case 6: return launch<Form<2, true, 1>>(mk, mv, p, s, st);
    default: return launch<Form<2, true, 2>>(mk, mv, p, s, st);
  }
}

B2_DEFINE_STATUS(treeattn)
