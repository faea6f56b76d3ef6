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
// A CTA, one to an SM: two warps copy (tiled TMA, 16 keys x 64 dims a box, 128-byte swizzle; pages behind the end are asked for outside the tensor and
// come as zeros), one issues the products for scores and one those of P V, each waiting for a ring's places in their order (a parity wait that could be
// more than one phase ahead would return at once); two groups of 256 threads do softmax, four threads to two query rows of a
// tile's 64 keys.  Scores come from tensor memory into registers once, and their place is free for the next ones; P goes back to tensor memory
// as the A operand of P V; the accumulator is rescaled only where a row's maximum grew by more than 2^6.
//   up to 128 query rows (NW 1): both groups have the same rows and take every other tile, each with its own maxima, sums and accumulator, which
//     meet at the segment's end; the queries are in tensor memory.  One softmax takes longer than its tile's bytes, two at a time do not.
//   up to 256 (NW 2): a group has a query tile of its own and both share every K / V tile; the queries are in shared memory.
// More rows take further CTAs (blockIdx.y) over the same keys.
// An 8-bit cache comes in as bytes (bulk copies, scales with them); four warps for keys and four for values make b / 64 in bf16 of them, which is
// exact; K's scale goes on the scores and V's on the weights, both in fp32.  Of four dimensions the second and the third change places on the way (pairs come apart that
// way), which the queries follow and the results undo.
//
// What bounds it (times of twenty calls in a graph; in long streams of calls the power cap adds a tenth and more to the large ones).  bf16 with one query
// tile: the cache's bytes (32 requests of 2000 to 33000 positions, 40 heads on 8 of 128: 2.3 GB in 383 us, 6.0 TB/s of the 6.5 that a copy reaches; 424 in a
// stream).  Two query tiles: the softmax, a chain of about 2000 cycles a tile whose four warps to a scheduler hide half of it, and the scores' product, which
// reads Q from shared memory (16 requests of up to 9000 positions, 40 to 64 nodes, 16 heads on 4: 173 MB in 66 us).  8 bits: instructions, 4600 a tile in 71 % of
// the issue slots, of which the expansion is about 800 and the arithmetic of the scores about 1200 by the code; the rest, 140 bytes of spills
// in it, has not been taken apart (12 requests of up to 65000 positions, 24 nodes, 40 heads on 8: 1.09 GB in 404 us; 471 in a stream).  One request: a segment's
// start and end, about four tiles' time, and the second launch (4100 positions: 18 us).  Full tables of many short requests: the same, a request at a time.
#include "tree.cuh"

using namespace b2;

namespace {

constexpr int kPage = kTreePage, kMaxNodes = kTreeNodes, kMaxReq = kTreeRequests;
constexpr int BQ = 128, BK = 64;
constexpr int kScales = 8;       // tiles whose scales are kept
constexpr int kKept = 256;       // requests whose lengths and rows are kept in shared memory

struct TreeAttnParams {
  const __nv_bfloat16* q;
  long long ldq;
  const int8_t *k8, *v8;           // 8-bit form
  const float *k_scale, *v_scale;
  const int *lengths, *row_start, *row_pos, *block_table, *tree_table;
  const unsigned long long* masks;
  int B, max_blocks, tree_blocks, num_pages, rows, n_q, n_kv, gqa, window;
  int group_tokens;                // nodes to a CTA's query tiles
  int single;                      // > 0: places of a request's key head, each a column of its own
  float scale_log2;
  __nv_bfloat16* out;
  long long ldo;
  float *part_o, *part_ml;         // [group][column][2][D / 4][NW x 128 rows][4], and [...][rows] maximum and sum
  int* sched;                      // places a column, the requests' first places (of one key head), their tiles
};

template <int NDK_, bool I8_, int NW_>
struct Form {
  static constexpr int NDK = NDK_, NW = NW_, D = NDK_ * 64;
  static constexpr bool I8 = I8_;
  static constexpr int T_BYTES = BK * NDK * 128;                 // a K or V tile: [64-dim blocks][64 keys][128 bytes]
  static constexpr int KS = I8_ ? (NW_ == 1 ? 3 : 2) : (NW_ == 1 ? 6 : 4) * (3 - NDK_), VS = I8_ ? (NW_ == 1 ? 3 : 2) : (NW_ == 1 ? 7 : 5) * (3 - NDK_);     // operand tiles
  static constexpr int RS = I8_ ? (NW_ == 1 ? 5 : 4) * (3 - NDK_) : 0;                                                     // stages of bytes
  static constexpr int S_BYTES = 2 * BK * D + 2 * BK * 4;        // keys, values, their scales
  static constexpr int Q_BYTES = NW == 1 ? 0 : NW * BQ * NDK * 128;
  static constexpr int kMma = 2, kSoft = 4, kConv = kSoft + 16, kConvThreads = 256, kWarps = kConv + (I8_ ? kConvThreads / 32 : 0), kThreads = kWarps * 32;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + KS * T_BYTES, OFF_ST = OFF_V + VS * T_BYTES, OFF_SC = OFF_ST + RS * S_BYTES,
                       OFF_X = OFF_SC + (I8_ ? kScales * 2 * BK * 4 : 0), OFF_CUM = OFF_X + 2 * 2 * BQ * 4, OFF_REQ = OFF_CUM + (kMaxReq + 8) * 4, OFF_BAR = OFF_REQ + 3 * kKept * 4,
                       SMEM = OFF_BAR + 1024 + 1024;
  static_assert(SMEM <= 227 * 1024 && KS <= 14 && VS <= 14 && RS <= 14, "shared memory");
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

// columns of the thread's row between registers and tensor memory
__device__ __forceinline__ void st_16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
               : "memory");
}
// 16 rows x 64 columns: the thread has rows t / 4 (registers 4 b, 4 b + 1) and t / 4 + 8 (4 b + 2, 4 b + 3), columns 8 b + 2 (t % 4) and the next
#define TREE_LD_16x64(taddr, r)                                                                                                      \
  asm volatile(                                                                                                                      \
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "                                                                                      \
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, "    \
      "[%32];"                                                                                                                       \
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),       \
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),          \
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),          \
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])                                                                           \
      : "r"(taddr)                                                                                                                   \
      : "memory")
#define TREE_ST_16x64(taddr, r)                                                                                                      \
  asm volatile(                                                                                                                      \
      "tcgen05.st.sync.aligned.16x256b.x8.b32 [%32], "                                                                               \
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::  \
          "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),   \
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),         \
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),         \
      "r"(r[31]), "r"(taddr)                                                                                                         \
      : "memory")
// 16 rows x 32 columns: rows t / 4 (register 2 b) and t / 4 + 8 (2 b + 1), column 4 b + t % 4
__device__ __forceinline__ void st_16x32(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void st_8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void ld_16(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                 "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
// Bounded waits of a whole warp.  The vote is inside the loop: a warp never comes apart at a wait, which everything behind it that is a warp's
// (tensor memory, named barriers, operands in uniform registers) takes for granted.
__device__ __forceinline__ bool warp_wait_inline(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 256; ++i)
    if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
  const long long t0 = clock64();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
    if (__any_sync(0xffffffffu, clock64() - t0 > kWaitCycles)) {
      if ((threadIdx.x & 31) == 0) record_error(ERR_ATTN_WAIT, (blockIdx.x << 8) | (threadIdx.x >> 5));
      __syncwarp();
      return false;
    }
  }
}
__device__ __noinline__ bool warp_wait_long(uint32_t bar, uint32_t parity) { return warp_wait_inline(bar, parity); }
// The first look inline, for warps whose phase usually is over; the call is the whole warp's.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, ok != 0) || warp_wait_long(bar, parity);
}
// One lane of a warp that is together.  The issuing warps stay together around it, with every operand the same in all lanes, so that operands are
// in uniform registers: a lone lane pays for moving each of them there.
__device__ __forceinline__ bool elect() {
  __syncwarp();
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}
__device__ __forceinline__ void ld_shared(uint32_t at, uint32_t* r) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
// One arrival for a warp: 32 lanes that arrive at one barrier are served one after another.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Four bytes, their sign bits turned over (u = b + 128), as bf16 pairs b / 64: up to 255 the bits of a bf16 are an integer times 2^-133 (subnormal
// or not), so one multiply-add makes u 2^-133 2^127 - 2 = (u - 128) / 64.  Three logic instructions a word; the logic pipe is what the expansion of
// an 8-bit cache is bound by (with a mantissa trick for either sign, nine: 404 cycles for 8 KB, more than their way from HBM).
__device__ __forceinline__ uint32_t scaled_bf16(uint32_t pair) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(pair), "r"(0x7f007f00u), "r"(0xc000c000u));
  return d;
}
constexpr float kByteScale = 64.f;      // what the scales make good

// Zeros for what is no number in the first rows of a tile of values: a lane's first piece of 16 bytes, further ones 32 pieces on.
template <int NDK>
__device__ __noinline__ void zero_no_numbers(uint32_t at, int rows) {
  const int lane = threadIdx.x & 31;
  for (int x = lane; x < rows * (NDK * 8); x += 32) {
    const uint32_t to = at + (x - lane) * (16 / NDK);
    uint32_t u[4];
    ld_shared(to, u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if ((u[e] & 0x7f80u) == 0x7f80u) u[e] &= 0xffff0000u;
      if ((u[e] & 0x7f800000u) == 0x7f800000u) u[e] &= 0xffffu;
    }
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
  }
  fence_proxy_async_smem();
}

// The weight of a part of a row's keys whose maximum is m beside others' of up to `best`: 0 only where the row saw nothing of the part (what such a part
// holds is not looked at), else 2^-126 at least.  That is nothing beside a sum of numbers, but leaves a part that is no number what it is, wherever the
// row's keys were cut (a weight of 0 in 32 bits would drop it or make it NaN).
__device__ __forceinline__ float part_weight(float m, float best) { return m == -INFINITY ? 0.f : fmaxf(exp2f(m - best), 1.17549435e-38f); }

// A request as the roles see it.
struct Req {
  int b, r0, n, length, first, nt;      // first row, nodes, cached positions, first tile of the cache that is read, tiles (the tree's is the last)
};

__device__ __forceinline__ int first_tile(const TreeAttnParams& p, int length) { return p.window > 0 ? max(0, length - p.window + 1) / BK : 0; }
__device__ __forceinline__ int tiles_of(const TreeAttnParams& p, int length) { return (length + BK - 1) / BK - first_tile(p, length) + 1; }
__device__ __forceinline__ int length_of(const TreeAttnParams& p, int b) { return max(0, min(p.lengths[b], p.max_blocks * kPage)); }
__device__ __forceinline__ int nodes_of(const TreeAttnParams& p, int b, int& r0) {
  r0 = p.row_start[b];
  return max(0, min(min(p.row_start[b + 1], p.rows) - r0, kMaxNodes));
}

// The segments of a CTA's part [u, u1) of the line of tiles.  A request's tiles of one key head take s_cum[b + 1] - s_cum[b] places of it.
struct Walk {
  int u, u0, u1, b;
  Req r;
  int h, ts, count, tok;       // key head, first tile and tiles of the segment, nodes of the CTA's group
};

__device__ __forceinline__ void begin_walk(const TreeAttnParams& p, const int* s_cum, int total, int each, Walk& k) {
  k.u0 = k.u = min(total, (int)blockIdx.x * each);
  k.u1 = min(total, k.u0 + each);
  int lo = 0, hi = p.B - 1;      // the last request that begins at or before u0
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_cum[mid] * p.n_kv <= k.u0) lo = mid; else hi = mid - 1;
  }
  k.b = lo;
}

// s_req: tiles, cached positions and first row of up to kKept requests
template <class F>
__device__ __forceinline__ bool next_segment(const TreeAttnParams& p, const int* s_cum, const int* s_req, Walk& k) {
  for (;;) {
    if (k.u >= k.u1) return false;
    while (s_cum[k.b + 1] * p.n_kv <= k.u) ++k.b;
    const int places = s_cum[k.b + 1] - s_cum[k.b], rel = k.u - s_cum[k.b] * p.n_kv;
    k.h = rel / places;
    k.ts = rel - k.h * places;
    k.r.b = k.b;
    if (p.B <= kKept) {
      k.r.length = s_req[kKept + k.b];
      const int rn = s_req[2 * kKept + k.b];
      k.r.r0 = rn >> 7;
      k.r.n = rn & 127;
    } else {
      k.r.n = nodes_of(p, k.b, k.r.r0);
      k.r.length = length_of(p, k.b);
    }
    k.r.first = first_tile(p, k.r.length);
    k.r.nt = tiles_of(p, k.r.length);
    if (k.ts >= k.r.nt) {      // places behind the last tile
      k.u += places - k.ts;
      continue;
    }
    k.count = min(k.r.nt - k.ts, k.u1 - k.u);
    k.u += k.count;
    k.tok = min(p.group_tokens, k.r.n - (int)blockIdx.y * p.group_tokens);
    if (k.tok > 0) return true;
  }
}

// Tiles that some rows may see less of than others: the tree's, and with a window those that it begins in for any of the tree's rows.
__device__ __forceinline__ bool uneven(const TreeAttnParams& p, const Req& r, int t) {
  return t == r.nt - 1 || (p.window > 0 && (r.first + t) * BK < r.length + r.n - p.window);
}

// Values that are no numbers, in uneven tiles: a product with a weight of 0 would give them to rows that do not see them, so such a tile has zeros
// there, and where that was so the CTA goes through its segments once more when all is done, and adds them to the results (or partial sums) of the
// rows that see them.  Such a value decides its sum whatever its weight is.
template <class F>
__device__ __noinline__ void add_no_numbers(const TreeAttnParams& p, const int* s_cum, const int* s_req, int each) {
  constexpr int C = 8, D = F::D, R = F::NW * BQ;
  Walk k;
  begin_walk(p, s_cum, s_cum[p.B] * p.n_kv, each, k);
  while (next_segment<F>(p, s_cum, s_req, k)) {
    const Req& r = k.r;
    for (int item = threadIdx.x; item < k.tok * p.gqa * (D / C); item += F::kThreads) {
      const int rr = item / (D / C), c0 = item % (D / C) * C, row = r.r0 + (int)blockIdx.y * p.group_tokens + rr / p.gqa, head = k.h * p.gqa + rr % p.gqa;
      const int lo = p.window > 0 ? p.row_pos[row] - p.window + 1 : 0;
      const unsigned long long mask = p.masks[row];
      float more[C] = {};
      for (int t = k.ts; t < k.ts + k.count; ++t) {
        if (!uneven(p, r, t)) continue;
        const bool tree = t == r.nt - 1;
        const int key0 = (r.first + t) * BK, keys = tree ? r.n : min(BK, r.length - key0);
        for (int x = 0; x < keys; ++x) {
          const int i = (tree ? x : key0 + x) / kPage;
          if (tree ? !(mask >> x & 1) || (p.window > 0 && p.row_pos[r.r0 + x] < lo) : key0 + x < lo) continue;
          int page = tree ? i < p.tree_blocks ? p.tree_table[(size_t)r.b * p.tree_blocks + i] : 0 : p.block_table[(size_t)r.b * p.max_blocks + i];
          if (page < 0 || page >= p.num_pages) page = 0;
          const long long at = ((long long)page * p.n_kv + k.h) * kPage + x % kPage;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            float f;
            if (F::I8) f = (float)p.v8[at * D + c0 + c] * p.v_scale[at];
            else f = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.v8)[at * D + c0 + c]);
            if (f - f != 0.f) more[c] += f;
          }
        }
      }
      const size_t slot = (((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + (k.u - k.count != k.u0)) * R;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (more[c] == 0.f) continue;
        __nv_bfloat16* o = p.out + row * p.ldo + head * D + c0 + c;
        if (k.count == r.nt) *o = __float2bfloat16(__bfloat162float(*o) + more[c]);
        else p.part_o[slot * D + (size_t)((c0 + c) / 4) * (R * 4) + rr * 4 + (c & 3)] += more[c];
      }
    }
  }
}

template <class F>
__global__ void __launch_bounds__(F::kThreads, 1)
tree_attn_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TreeAttnParams p) {
  constexpr int NDK = F::NDK, NW = F::NW, KS = F::KS, VS = F::VS, D = F::D, RS = F::I8 ? F::RS : 1;
  constexpr int kStep = NW == 1 ? 2 : 1;      // a group's next tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_s = base, k_s0 = base + F::OFF_K, v_s0 = base + F::OFF_V, st_s0 = base + F::OFF_ST, bars = base + F::OFF_BAR;
  int* const s_cum = reinterpret_cast<int*>(gen + F::OFF_CUM);
  int* const s_req = reinterpret_cast<int*>(gen + F::OFF_REQ);
  float* const s_scale = reinterpret_cast<float*>(gen + F::OFF_SC);       // [kScales][K, V][64]
  float* const s_x = reinterpret_cast<float*>(gen + F::OFF_X);            // [group][maximum, sum][128]
  const uint32_t b_kfull = bars, b_kempty = bars + 112, b_vfull = bars + 224, b_vempty = bars + 336, b_rfull = bars + 448, b_rempty = bars + 560, b_q = bars + 672;
  auto b_sfull = [&](int w) { return bars + 680 + w * 8; };
  auto b_sfree = [&](int w) { return bars + 696 + w * 8; };
  auto b_pfull = [&](int w) { return bars + 712 + w * 8; };
  auto b_odone = [&](int w) { return bars + 728 + w * 8; };
  auto b_scale = [&](int g) { return bars + 744 + (g % kScales) * 8; };
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(gen + F::OFF_BAR + 808);
  int* const s_sums = reinterpret_cast<int*>(gen + F::OFF_BAR + 816);      // [32], [8]
  volatile int* const s_odd = s_sums + 40;         // an uneven tile had values that are no numbers; places a column
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (tid == 0) *s_odd = 0;
  if (tid == 0) {
    for (int i = 0; i < KS; ++i) {
      mbar_init(b_kfull + 8 * i, F::I8 ? F::kConvThreads / 64 : 1);
      mbar_init(b_kempty + 8 * i, 1);
    }
    for (int i = 0; i < VS; ++i) {
      mbar_init(b_vfull + 8 * i, F::I8 ? F::kConvThreads / 64 : 1);
      mbar_init(b_vempty + 8 * i, 1);
    }
    if (F::I8) {
      for (int i = 0; i < RS; ++i) {
        mbar_init(b_rfull + 8 * i, 2);
        mbar_init(b_rempty + 8 * i, F::kConvThreads / 32);
      }
      for (int i = 0; i < kScales; ++i) mbar_init(b_scale(i), 4);
    }
    mbar_init(b_q, 16);
    for (int w = 0; w < 2; ++w) {
      mbar_init(b_sfull(w), 1);
      mbar_init(b_sfree(w), 8);
      mbar_init(b_pfull(w), 8);
      mbar_init(b_odone(w), 1);
    }
    mbar_fence_init();
    if (!F::I8) {
      prefetch_tmap(&map_k);
      prefetch_tmap(&map_v);
    }
  }
  if (warp == F::kMma) {
    __syncwarp();
    tmem_alloc(smem_u32(tmem_slot), 512);
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
      const int length = length_of(p, b), n = nodes_of(p, b, r0);
      const int nt = n > 0 ? tiles_of(p, length) : 0;
      s_cum[b + 1] = mine += nt;
      if (b < kKept) {
        s_req[b] = nt;
        s_req[kKept + b] = length;
        s_req[2 * kKept + b] = r0 << 7 | n;
      }
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
    if (b0 < p.B)
      for (int w = 0; w < warp; ++w) before += s_sums[w];
    for (int b = b0; b < min(b0 + per, p.B); ++b) s_cum[b + 1] += before;
    if (tid == 0) s_cum[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  // tensor memory: queries 64 columns (NW 1), scores 2 x 64, weights 2 x 32, accumulators 2 x D
  const uint32_t t_q = tmem_base;
  auto t_s = [&](int w) { return tmem_base + 64 + (uint32_t)w * 64; };
  auto t_p = [&](int w) { return tmem_base + 192 + (uint32_t)w * 32; };
  auto t_o = [&](int w) { return tmem_base + 256 + (uint32_t)w * D; };

  int total = s_cum[p.B] * p.n_kv, each = p.single ? p.single : (total + gridDim.x - 1) / gridDim.x;
  // Where there are columns enough for every request's key head, a request's tiles can begin a column: then a CTA has one segment, whose start and
  // end cost as much as four or five tiles.  Eight column lengths from the least on are looked at; the first that fits is taken.
  // (One request of 4100 positions, 8 key heads, 66 tiles: 17 columns of 4 instead of 16.5; 21.2 -> 16.7 us with the merge, before values were looked at, 18.0 now.)
  // single: tables so short that a request's key head is one column in any case, and nothing is left to merge.
  if (p.single || p.B * p.n_kv <= (int)gridDim.x) {
    if (warp == 0) {
      bool fits = p.single > 0;
      if (!fits && each > 0) {      // lanes: eight lengths x four parts of the requests
        const int len = each + (lane & 7);
        int sum = 0;
        for (int b = lane >> 3; b < p.B; b += 4) sum += (s_req[b] + len - 1) / len;
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const unsigned good = __ballot_sync(0xffffffffu, sum * p.n_kv <= (int)gridDim.x) & 0xff;
        fits = good != 0;
        if (fits) each += __ffs(good) - 1;
      }
      if (fits && each > 0) {      // the line again, in whole columns
        int before = 0;
#pragma unroll 1
        for (int b0 = 0; b0 < p.B; b0 += 32) {
          const int b = b0 + lane;
          int r0, nt = 0;
          if (b < p.B) nt = p.single ? (nodes_of(p, b, r0) > 0 ? 1 : 0) : s_req[b];
          int x = (nt + each - 1) / each * each;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
          }
          if (b < p.B) s_cum[b + 1] = before + x;
          before += __shfl_sync(0xffffffffu, x, 31);
        }
      }
      if (lane == 0) s_sums[32] = each;
    }
    __syncthreads();
    each = s_sums[32];
    total = s_cum[p.B] * p.n_kv;
  }
  if (!p.single && blockIdx.x == 0 && blockIdx.y == 0) {
    for (int b = tid; b <= p.B; b += F::kThreads) {
      p.sched[b + 1] = s_cum[b];
      if (b < p.B) {
        int r0;
        p.sched[p.B + 2 + b] = p.B <= kKept ? s_req[b] : nodes_of(p, b, r0) > 0 ? tiles_of(p, length_of(p, b)) : 0;
      }
    }
    if (tid == 0) p.sched[0] = each;
  }
  if (tid == 0) s_odd[1] = each;
  Walk k;
  begin_walk(p, s_cum, total, each, k);
  // keys of tile t of the walk's request
  auto keys_of = [&](int t) { return t == k.r.nt - 1 ? k.r.n : min(BK, k.r.length - (k.r.first + t) * BK); };

  if (warp < F::kMma) {
    // ---------------------------------------------------------- copies of keys (warp 0) and of values (warp 1): page numbers in the lanes, one
    // thread issues (eight lanes that issue a box each are served one after another: 1850 cycles for a tile's 16 boxes)
    bool ok = true;
    int g = 0;
    const bool is_v = warp == 1;
    const int kd = F::I8 ? RS : is_v ? VS : KS;      // depth of this warp's ring
    const uint32_t full0 = F::I8 ? b_rfull : is_v ? b_vfull : b_kfull, empty0 = F::I8 ? b_rempty : is_v ? b_vempty : b_kempty;
    int s = 0, par = 0;
    while (ok && next_segment<F>(p, s_cum, s_req, k)) {
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
        int page[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) page[x] = __shfl_sync(0xffffffffu, tree ? tree_ids : ids, tree ? x : pi - at + x);
        if (g >= kd) ok = warp_wait_inline(empty0 + 8 * s, par ^ 1);
        if (!ok) break;
        const uint32_t full = full0 + 8 * s;
        if constexpr (F::I8) {
          if (elect()) {
            int pages = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) pages += page[x] >= 0;
            mbar_expect_tx(full, pages * (kPage * D + kPage * 4));
            const uint32_t st = st_s0 + s * F::S_BYTES + (is_v ? BK * D : 0), sc = st_s0 + s * F::S_BYTES + 2 * BK * D + (is_v ? BK * 4 : 0);
            const int8_t* data = is_v ? p.v8 : p.k8;
            const float* scale = is_v ? p.v_scale : p.k_scale;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (page[x] >= 0) {
                const long long row = ((long long)page[x] * p.n_kv + k.h) * kPage;
                bulk_g2s(st + x * (kPage * D), data + row * D, kPage * D, full);
                bulk_g2s(sc + x * (kPage * 4), scale + row, kPage * 4, full);
              }
          }
        } else {
          const uint32_t dst = (is_v ? v_s0 : k_s0) + s * F::T_BYTES;
          const CUtensorMap* map = is_v ? &map_v : &map_k;
          if (elect()) {
            mbar_expect_tx(full, F::T_BYTES);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int row = (page[x] >= 0 ? page[x] * p.n_kv + k.h : p.num_pages * p.n_kv) * kPage;
#pragma unroll
              for (int c = 0; c < NDK; ++c) tma_load_2d(dst + c * (BK * 128) + x * (kPage * 128), map, c * 64, row, full);
            }
          }
        }
        __syncwarp();
        if (++s == kd) { s = 0; par ^= 1; }
      }
    }
    if (!ok)      // copies in flight end before the CTA does
      for (int i = max(0, g - kd); i < g; ++i) warp_wait_inline(full0 + 8 * (i % kd), (i / kd) & 1);
  } else if (warp == F::kMma) {
    // ---------------------------------------------------------- scores: S = Q K^T of every tile, as its keys come and its group's place is free
    constexpr uint32_t idesc_qk = make_idesc(1, 1, BQ, BK);
    const uint32_t hi_k = (uint32_t)(make_desc_sw128(0) >> 32);
    const uint32_t q_lo = (uint32_t)make_desc_sw128(q_s), k_lo = (uint32_t)make_desc_sw128(k_s0);
    bool ok = true;
    int g = 0, seg = 0, ks = 0, par = 0, j[2] = {0, 0};      // tiles so far, of all and of either group
    while (ok && next_segment<F>(p, s_cum, s_req, k)) {
      ok = warp_wait_inline(b_q, seg & 1);
      for (int i = 0; i < k.count && ok; ++i, ++g) {
        ok = warp_wait_inline(b_kfull + 8 * ks, par);
        const uint32_t kl = k_lo + ks * (F::T_BYTES >> 4);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (NW == 1 && w != (g & 1)) continue;
          if (ok && j[w] >= 1) ok = warp_wait_inline(b_sfree(w), (j[w] - 1) & 1);      // the scores before are in registers
          if (!ok) break;
          ++j[w];
          const bool live = NW == 1 || w * BQ < k.tok * p.gqa;      // (a second query tile without rows only hands tiles back)
          tc_fence_after();
          if (elect()) {
            if (live) {
#pragma unroll
              for (int x = 0; x < 4 * NDK; ++x) {
                const uint32_t kx = kl + (((x >> 2) * (BK * 128) + (x & 3) * 32) >> 4);
                if constexpr (NW == 1) umma_f16_ts_w(t_s(w), t_q + 8 * x, kx, hi_k, idesc_qk, x != 0);
                else umma_f16_w(t_s(w), q_lo + ((w * (BQ * NDK * 128) + (x >> 2) * (BQ * 128) + (x & 3) * 32) >> 4), hi_k, kx, hi_k, idesc_qk, x != 0);
              }
            }
            tc_commit(b_sfull(w));
            if (NW == 1 || w == 1) tc_commit(b_kempty + 8 * ks);
          }
          __syncwarp();
        }
        if (++ks == KS) { ks = 0; par ^= 1; }
      }
      ++seg;
    }
  } else if (warp < F::kSoft) {
    // ---------------------------------------------------------- results: O += P V
    constexpr uint32_t idesc_pv = make_idesc(1, 1, BQ, D) | (1u << 16);      // V is MN-major
    const uint32_t hi_v = (uint32_t)(make_desc_v(0) >> 32), v_lo = (uint32_t)make_desc_v(v_s0);
    bool ok = true;
    int g = 0, vs = 0, par = 0, j[2] = {0, 0};
    while (ok && next_segment<F>(p, s_cum, s_req, k)) {
      for (int i = 0; i < k.count && ok; ++i, ++g) {
        const int valid = keys_of(k.ts + i);
        ok = warp_wait_inline(b_vfull + 8 * vs, par);
        if (!F::I8 && ok && (valid & 15) != 0) {
          // values behind the last key's are anything: their weights are 0, but 0 x infinity is not
          const int end = (valid + 15) & ~15;
          for (int x = lane; x < (end - valid) * NDK * 8; x += 32) {
            const int row = valid + x / (NDK * 8), c = x % (NDK * 8);
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(v_s0 + vs * F::T_BYTES + (c >> 3) * (BK * 128) + row * 128 + (c & 7) * 16), "r"(0) : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (!F::I8 && ok && uneven(p, k.r, k.ts + i)) {
          // x 0 is 0 of numbers alone.  Two pieces at a time: the warp comes here once a segment, and the way of
          // so many instructions to it is what the look costs (128 requests of 16 tiles: 110 us without it, 111, 112, 114, 118 with 1, 2, 4, 8
          // pieces; 16 of 6 tiles 10.5; 11.0, 10.9, 10.8, 10.8).
          const uint32_t at = v_s0 + vs * F::T_BYTES + (lane & (NDK - 1)) * (BK * 128) + (lane >> (NDK - 1)) * 16;
          uint32_t zero = 0;
#pragma unroll 2
          for (int x = lane; x < valid * (NDK * 8); x += 32) {
            uint32_t u[4];
            ld_shared(at + (x - lane) * (16 / NDK), u);
#pragma unroll
            for (int e = 0; e < 4; ++e) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(zero) : "r"(u[e]), "r"(0));
          }
          if (__any_sync(0xffffffffu, (zero & 0x7fff7fffu) != 0)) {
            zero_no_numbers<NDK>(at, valid);
            *s_odd = 1;
          }
          __syncwarp();
        }
        const uint32_t vl = v_lo + vs * (F::T_BYTES >> 4);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (NW == 1 && w != (g & 1)) continue;
          if (ok) ok = warp_wait_inline(b_pfull(w), j[w] & 1);
          if (!ok) break;
          ++j[w];
          const bool live = NW == 1 || w * BQ < k.tok * p.gqa;
          const bool first = i < kStep;      // the group's first tile of the segment
          tc_fence_after();
          if (elect()) {
            if (live) {
#pragma unroll
              for (int x = 0; x < 4; ++x)      // 16 keys a step; P in tensor memory, 8 columns of pairs
                umma_f16_ts_w(t_o(w), t_p(w) + 8 * x, vl + ((x * 16 * 128) >> 4), hi_v, idesc_pv, !first || x != 0);
            }
            tc_commit(b_odone(w));
            if (NW == 1 || w == 1) tc_commit(b_vempty + 8 * vs);
          }
          __syncwarp();
        }
        if (++vs == VS) { vs = 0; par ^= 1; }
      }
    }
    // the last arrival that a product makes: none is on its way when the CTA ends
    if (ok && g > 0) warp_wait_inline(b_vempty + 8 * ((g - 1) % VS), ((g - 1) / VS) & 1);
  } else if (warp < F::kConv) {
    // ---------------------------------------------------------- softmax: two threads per query row of group w
    constexpr float kLazy = 6.f;
    const int sw = warp - F::kSoft, w = sw >> 3, half = (sw >> 2) & 1, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    // scores: 16 rows of the quarter's 32 to a warp, half a row's 64 columns to four threads that pass maxima on by shuffles (with the
    // columns cut between two warps they had to meet at a barrier in every tile); queries and results: a row to a lane, columns cut
    const int mr = quarter * 32 + half * 16 + (lane >> 2), mc = 2 * (lane & 3);      // this thread's rows mr and mr + 8, its first column
    const uint32_t half_addr = (uint32_t)(quarter * 32 + half * 16) << 16;
    // once a wait has run out no other is made, but every barrier is still come to
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (ok) ok = warp_wait(bar, parity);
    };
    int g0 = 0, j = 0, seg = 0;
    while (next_segment<F>(p, s_cum, s_req, k)) {
      const int rr = (NW == 1 ? 0 : w * BQ) + r, live_rows = k.tok * p.gqa;
      const bool row_ok = rr < live_rows, warp_ok = rr - lane < live_rows;
      const int node = blockIdx.y * p.group_tokens + rr / p.gqa, head = k.h * p.gqa + rr % p.gqa, row = k.r.r0 + node;
      // ---- the queries: the products of the segment before are done, all threads came by its end
      {
        constexpr int NV = NW == 1 ? D / 32 : D / 16;      // pieces of 8 dims that this thread brings: a quarter of its row, or half
        const int c0 = NW == 1 ? (w * 2 + half) * NV : half * NV;
        uint4 x[NV] = {};
        if (row_ok) {
          const uint4* src = reinterpret_cast<const uint4*>(p.q + row * p.ldq + head * D) + c0;
#pragma unroll
          for (int c = 0; c < NV; ++c) x[c] = src[c];
        }
        if constexpr (F::I8) {
#pragma unroll
          for (int c = 0; c < NV; ++c)
            x[c] = make_uint4(__byte_perm(x[c].x, x[c].y, 0x5410), __byte_perm(x[c].x, x[c].y, 0x7632), __byte_perm(x[c].z, x[c].w, 0x5410), __byte_perm(x[c].z, x[c].w, 0x7632));
        }
        if constexpr (NW == 1) {
          __syncwarp();      // (tensor memory is a whole warp's: lanes whose ways parted meet again first, here and below)
          if constexpr (NV == 4) st_16(t_q + lane_addr + c0 * 4, reinterpret_cast<const uint32_t*>(x));
          else st_8(t_q + lane_addr + c0 * 4, reinterpret_cast<const uint32_t*>(x));
          tmem_st_wait();
          tc_fence_before();
        } else {
#pragma unroll
          for (int c = 0; c < NV; ++c)
            *reinterpret_cast<uint4*>(gen + w * (BQ * NDK * 128) + ((c0 + c) >> 3) * (BQ * 128) + r * 128 + ((((c0 + c) & 7) ^ (r & 7)) << 4)) = x[c];
          fence_proxy_async_smem();
        }
        warp_arrive(b_q);
      }
      wait(b_q, seg & 1);      // (all threads are done with the segment before)
      ++seg;
      const bool some = (NW == 1 ? 0 : w * BQ) + quarter * 32 + half * 16 < live_rows;      // rows of a request in this warp's scores
      int lo[2] = {0, 0};                            // the first position that is seen
      unsigned long long mask[2] = {0, 0};
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int qr = (NW == 1 ? 0 : w * BQ) + mr + 8 * y;
        if (qr >= live_rows) continue;
        const int at = k.r.r0 + blockIdx.y * p.group_tokens + qr / p.gqa;
        if (p.window > 0) lo[y] = p.row_pos[at] - p.window + 1;
        if (k.ts + k.count == k.r.nt) {
          mask[y] = p.masks[at];
          if (k.r.n < 64) mask[y] &= (1ull << k.r.n) - 1;
          if (lo[y] > k.r.length)
            for (int i = 0; i < k.r.n; ++i)
              if (p.row_pos[k.r.r0 + i] < lo[y]) mask[y] &= ~(1ull << i);
        }
      }
      // tiles that all of the warp's rows see all of: plain0 <= t < plain1
      const int plain1 = min(k.r.length / BK - k.r.first, k.r.nt - 1);
      const int plain0 = p.window > 0 ? (max(0, __reduce_max_sync(0xffffffffu, max(lo[0], lo[1]))) + BK - 1) / BK - k.r.first : 0;
      // the reference that scores are taken against, negative (0 before the first key: 2^s of a row without any is not used); sums of this thread's columns
      float mref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      unsigned long long nm2[2] = {0ull, 0ull};
      const int i0 = NW == 1 ? (w - g0) & 1 : 0;
      for (int i = i0; i < k.count; i += kStep, ++j) {
        const int g = g0 + i, t = k.ts + i;
        wait(b_sfull(w), j & 1);
        if (F::I8) wait(b_scale(g), (g / kScales) & 1);
        if (!some) {      // rows of nobody: the products take what is there
          warp_arrive(b_sfree(w));
          if (i != i0) wait(b_odone(w), (j - 1) & 1);
          warp_arrive(b_pfull(w));
          continue;
        }
        tc_fence_after();
        uint32_t v[32];
        __syncwarp();
        TREE_LD_16x64(t_s(w) + half_addr, v);
        tmem_ld_wait();
        tc_fence_before();
        warp_arrive(b_sfree(w));
        // v[4 c + 2 y + e]: row mr + 8 y, column 8 c + mc + e
        const float* sc = s_scale + (g % kScales) * (2 * BK) + mc;
        if constexpr (F::I8) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const unsigned long long f = *reinterpret_cast<const unsigned long long*>(sc + 8 * c);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              unsigned long long a;
              asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "r"(v[4 * c + 2 * y]), "r"(v[4 * c + 2 * y + 1]));
              asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a) : "l"(f));
              asm("mov.b64 {%0, %1}, %2;" : "=r"(v[4 * c + 2 * y]), "=r"(v[4 * c + 2 * y + 1]) : "l"(a));
            }
          }
        }
        if (t < plain0 || t >= plain1) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            unsigned long long vis = mask[y];
            if (t != k.r.nt - 1) {
              const int key0 = (k.r.first + t) * BK, end = min(BK, k.r.length - key0), begin = lo[y] - key0;
              vis = end >= BK ? ~0ull : (1ull << end) - 1;
              vis = begin <= 0 ? vis : begin >= BK ? 0ull : vis & (~0ull << begin);
            }
            vis >>= mc;
            const uint32_t part[2] = {(uint32_t)vis, (uint32_t)(vis >> 32)};
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (!(part[c >> 2] >> (8 * (c & 3) + e) & 1)) v[4 * c + 2 * y + e] = 0xff800000u;
          }
        }
        const float factor = F::I8 ? 1.f : p.scale_log2;
        float top[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          top[y] = fmaxf(__uint_as_float(v[2 * y]), __uint_as_float(v[2 * y + 1]));
#pragma unroll
          for (int c = 1; c < 8; ++c) asm("max.f32 %0, %0, %1, %2;" : "+f"(top[y]) : "f"(__uint_as_float(v[4 * c + 2 * y])), "f"(__uint_as_float(v[4 * c + 2 * y + 1])));
        }
        top[0] *= factor;
        top[1] *= factor;
        // A row whose maximum grew by more than 2^kLazy gets a new reference: rare, and all of the warp goes that way.  (Only there do a row's four
        // threads ask one another.)
        const bool grown = __any_sync(0xffffffffu, top[0] > mref[0] + kLazy || top[1] > mref[1] + kLazy);
        float alpha[2] = {1.f, 1.f};
        if (grown) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            top[y] = fmaxf(top[y], __shfl_xor_sync(0xffffffffu, top[y], 1));
            top[y] = fmaxf(top[y], __shfl_xor_sync(0xffffffffu, top[y], 2));
            if (top[y] > mref[y] + kLazy) {
              alpha[y] = exp2f(mref[y] - top[y]);      // 0 at the row's first key
              mref[y] = top[y];
              l[y] *= alpha[y];
              asm("mov.b64 %0, {%1, %1};" : "=l"(nm2[y]) : "f"(-top[y]));
            }
          }
        }
        unsigned long long sc2, acc[2] = {0ull, 0ull};
        asm("mov.b64 %0, {%1, %1};" : "=l"(sc2) : "f"(factor));
        uint32_t pk[16];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          unsigned long long f = 0;
          if constexpr (F::I8) f = *reinterpret_cast<const unsigned long long*>(sc + BK + 8 * c);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            unsigned long long xy;
            asm("mov.b64 %0, {%1, %2};" : "=l"(xy) : "r"(v[4 * c + 2 * y]), "r"(v[4 * c + 2 * y + 1]));
            if (F::I8) asm("add.rn.f32x2 %0, %0, %1;" : "+l"(xy) : "l"(nm2[y]));
            else asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(xy) : "l"(sc2), "l"(nm2[y]));
            float x0, x1, e0, e1;
            asm("mov.b64 {%0, %1}, %2;" : "=f"(x0), "=f"(x1) : "l"(xy));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(x0));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(x1));
            unsigned long long ee;
            asm("mov.b64 %0, {%1, %2};" : "=l"(ee) : "f"(e0), "f"(e1));
            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc[y]) : "l"(ee));
            if constexpr (F::I8) {
              asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(ee) : "l"(f));
              asm("mov.b64 {%0, %1}, %2;" : "=f"(e0), "=f"(e1) : "l"(ee));
            }
            // (to bf16, since the product's operands are of one type, V's; the sum is of the weights as they were.  Results are 0.19 to 0.25 % from
            // those in 64 bits, 0.17 of it their own rounding)
            pk[2 * c + y] = pack_bf16(e0, e1);
          }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float a0, a1;
          asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(acc[y]));
          l[y] += a0 + a1;
        }
        if (i != i0) {      // the product before has read its weights, and the accumulator is whole
          wait(b_odone(w), (j - 1) & 1);
          tc_fence_after();
          if (grown) {
#pragma unroll 1
            for (int c = 0; c < NDK; ++c) {
              __syncwarp();
              TREE_LD_16x64(t_o(w) + half_addr + c * 64, v);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha[e >> 1 & 1]);
              TREE_ST_16x64(t_o(w) + half_addr + c * 64, v);
            }
          }
        }
        __syncwarp();
        st_16x32(t_p(w) + half_addr, pk);
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(b_pfull(w));
      }
      // ---- the segment's sums, once its last product is done
      if (i0 < k.count) wait(b_odone(w), (j - 1) & 1);
      // maxima and sums of all rows, for the lanes that have the results (written anew behind the next segment's start, which all threads come to)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
        l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
        if (l[y] != l[y]) mref[y] = INFINITY;      // (no number as a score: what is made of the row is none either)
        if ((lane & 3) == 0) {
          s_x[(w * 2) * BQ + mr + 8 * y] = mref[y];
          s_x[(w * 2 + 1) * BQ + mr + 8 * y] = l[y];
        }
      }
      tc_fence_before();
      __syncwarp();
      asm volatile("bar.sync 9, 512;" ::: "memory");
      tc_fence_after();
      const bool whole = k.count == k.r.nt;
      const size_t slot = (((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + (k.u - k.count != k.u0)) * (NW * BQ) + rr;
      if (warp_ok) {
        float f0 = 1.f, f1 = 1.f, best = s_x[(w * 2) * BQ + r], sum = s_x[(w * 2 + 1) * BQ + r];
        if constexpr (NW == 1) {
          const float m0 = s_x[r], m1 = s_x[2 * BQ + r];
          best = fmaxf(m0, m1);
          f0 = part_weight(m0, best);
          f1 = part_weight(m1, best);
          sum = s_x[BQ + r] * f0 + s_x[3 * BQ + r] * f1;
        }
        const float inv = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
        constexpr int NC = NW == 1 ? NDK : 2 * NDK;      // pieces of 16 columns that this thread writes: a quarter of the row, or half
        const int c0 = NW == 1 ? (w * 2 + half) * NC * 16 : half * NC * 16;
        __nv_bfloat16* dst = p.out + row * p.ldo + head * D + c0;
        float* part = p.part_o + (slot - rr) * D + (size_t)(c0 / 4) * (NW * BQ * 4) + rr * 4;      // [D / 4][rows][4]: lanes next to one another
#pragma unroll 1
        for (int c = 0; c < NC; ++c) {
          uint32_t o[16], o1[16];
          __syncwarp();
          if constexpr (NW == 1) {
            ld_16(t_o(0) + lane_addr + c0 + c * 16, o);
            ld_16(t_o(1) + lane_addr + c0 + c * 16, o1);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = __float_as_uint(((f0 != 0.f ? f0 * __uint_as_float(o[e]) : 0.f) + (f1 != 0.f ? f1 * __uint_as_float(o1[e]) : 0.f)) * inv);
          } else {
            ld_16(t_o(w) + lane_addr + c0 + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
          }
          if constexpr (F::I8) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const uint32_t t2 = o[e + 1];
              o[e + 1] = o[e + 2];
              o[e + 2] = t2;
            }
          }
          if (row_ok && whole) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<uint4*>(dst + c * 16 + 8 * e) = make_uint4(
                  pack_bf16(__uint_as_float(o[8 * e]), __uint_as_float(o[8 * e + 1])), pack_bf16(__uint_as_float(o[8 * e + 2]), __uint_as_float(o[8 * e + 3])),
                  pack_bf16(__uint_as_float(o[8 * e + 4]), __uint_as_float(o[8 * e + 5])), pack_bf16(__uint_as_float(o[8 * e + 6]), __uint_as_float(o[8 * e + 7])));
          } else if (row_ok) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4*>(part + (size_t)(c * 4 + e) * (NW * BQ * 4)) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        if (!whole && row_ok && half == 0 && (NW == 2 || w == 0)) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(best, sum);
      }
      __syncwarp();
      tc_fence_before();
      g0 += k.count;
    }
  } else if constexpr (F::I8) {
    // ---------------------------------------------------------- bytes to bf16: four warps for keys, four for values; a thread's piece is 16 bytes of a key
    const int ct = (tid - F::kConv * 32) & 127;
    const bool is_v = warp >= F::kConv + 4;
    // Eight threads in a row take four pieces of a key's half (64 dims) and four of the other half of the next key: their loads, and their stores
    // to the swizzled tile, meet eight different groups of banks.  The second round takes the other halves.
    const int cl = ct & 3, odd = (ct >> 2) & 1, row = 2 * (ct >> 3) + odd;
    const uint32_t src0 = row * D + (NDK == 2 ? odd * 64 : 0) + cl * 16, dst0 = (NDK == 2 ? odd * (BK * 128) : 0) + row * 128 + (((2 * cl) ^ (row & 7)) << 4);
    const uint32_t full0 = is_v ? b_vfull : b_kfull, empty0 = is_v ? b_vempty : b_kempty, tile0 = is_v ? v_s0 : k_s0;
    constexpr int PL = F::KS;
    static_assert(!F::I8 || F::KS == F::VS, "places of keys and values");
    bool ok = true;
    int g = 0, rs = 0, rpar = 0, ps = 0, ppar = 1;
    while (ok && next_segment<F>(p, s_cum, s_req, k))
      for (int i = 0; i < k.count; ++i, ++g) {
        const uint32_t st = st_s0 + rs * F::S_BYTES + (is_v ? BK * D : 0), dst = tile0 + ps * F::T_BYTES;
        ok = warp_wait(b_rfull + 8 * rs, rpar);
        if (ok && g >= PL) ok = warp_wait(empty0 + 8 * ps, ppar);
        if (!ok) break;
        // the scales of tile g - kScales are read: this place came free with a product of tile g - PL, and those of a tile's scores wait for the
        // scores of the group's tile before to be in registers.  Behind the last key scales are anything, and made 0: what a place holds that nobody sees must
        // not reach a sum.
        static_assert(kScales >= F::KS + 4, "scales of tiles under way");
        if (ct < BK) {
          float f = *reinterpret_cast<const float*>(gen + F::OFF_ST + rs * F::S_BYTES + 2 * BK * D + (is_v ? BK * 4 : 0) + ct * 4);
          if (is_v && f - f != 0.f && ct < keys_of(k.ts + i) && uneven(p, k.r, k.ts + i)) {      // (add_no_numbers)
            f = 0.f;
            *s_odd = 1;
          }
          s_scale[(g % kScales) * (2 * BK) + (is_v ? BK : 0) + ct] = ct >= keys_of(k.ts + i) ? 0.f : f * (is_v ? kByteScale : p.scale_log2 * kByteScale);
          warp_arrive(b_scale(g));
        }
#pragma unroll
        for (int u = 0; u < 2 * NDK; ++u) {      // two halves of rows 0 to 31, of rows 32 to 63
          const int up = u & (NDK - 1), low = u / NDK;
          uint32_t ww[4], o[8];
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(ww[0]), "=r"(ww[1]), "=r"(ww[2]), "=r"(ww[3]) : "r"(st + (src0 ^ (up * 64)) + low * (32 * D)));
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t x = ww[y] ^ 0x80808080u;
            o[2 * y] = scaled_bf16(x & 0x00ff00ffu);
            o[2 * y + 1] = scaled_bf16(__byte_perm(x, 0u, 0x4341));
          }
          const uint32_t to = dst + (dst0 ^ (up * (BK * 128))) + low * (32 * 128);
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to ^ 16), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
        }
        fence_proxy_async_smem();
        warp_arrive(full0 + 8 * ps);
        warp_arrive(b_rempty + 8 * rs);
        if (++rs == RS) { rs = 0; rpar ^= 1; }
        if (++ps == PL) { ps = 0; ppar ^= 1; }
      }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == F::kMma) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  if (*s_odd) add_no_numbers<F>(p, s_cum, s_req, s_odd[1]);
}

// Segments of a request's key head, added up in the order of the keys: a CTA takes 32 query rows x 32 columns, a lane a row (partial sums stand with
// their rows next to one another for that), four segments' loads on their way together.  Bound by its launch and two ways to memory: 4 us behind one
// request of 17 segments.  (Two segments at a time in half the registers, which finds room beside a CTA of the attention: 18.0 -> 20.7 us; eight: no change.)
template <int D>
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeAttnParams p, int columns, int slot_rows, int groups) {
  constexpr int PARTS = D / 32;
  __shared__ uint32_t s_out[32][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int item = blockIdx.x, z = item % groups, h = item / groups % p.n_kv, b = item / groups / p.n_kv;
  const int rr0 = blockIdx.y / PARTS * 32, c0 = blockIdx.y % PARTS * 32;
  const int each = p.sched[0], before = p.sched[1 + b], places = p.sched[2 + b] - before, nt = p.sched[p.B + 2 + b];
  int r0;
  const int n = nodes_of(p, b, r0), rows = (min(p.group_tokens, n - z * p.group_tokens)) * p.gqa;
  if (nt < 1 || rr0 >= rows) return;
  const int a = before * p.n_kv + h * places, first = a / each, last = (a + nt - 1) / each;
  if (first == last) return;      // one segment: its CTA wrote the result
  const int rr = min(rr0 + lane, slot_rows - 1);
  auto slot = [&](int c) { return (((size_t)z * columns + c) * 2 + (a > c * each)) * slot_rows; };
  constexpr int U = 4;
  float best = -INFINITY, sum = 0.f, acc[2][4] = {};
  for (int c = first; c <= last; c += U) {
    float4 x[U][2];
    float2 ml[U];
#pragma unroll
    for (int y = 0; y < U; ++y) {
      ml[y] = make_float2(-INFINITY, 0.f);
      if (c + y <= last) {
        const size_t at = slot(c + y);
        ml[y] = *reinterpret_cast<const float2*>(p.part_ml + (at + rr) * 2);
        const float* src = p.part_o + at * D + (size_t)(c0 / 4 + 2 * warp) * (slot_rows * 4) + rr * 4;
        x[y][0] = *reinterpret_cast<const float4*>(src);
        x[y][1] = *reinterpret_cast<const float4*>(src + slot_rows * 4);
      }
    }
    float m = best;
#pragma unroll
    for (int y = 0; y < U; ++y) m = fmaxf(m, ml[y].x);
    const float old = part_weight(best, m);
    best = m;
    sum *= old;
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d >> 2][d & 3] *= old;
#pragma unroll
    for (int y = 0; y < U; ++y) {
      const float f = part_weight(ml[y].x, best);
      if (f != 0.f) {
        sum += f * ml[y].y;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          acc[e][0] += f * x[y][e].x; acc[e][1] += f * x[y][e].y; acc[e][2] += f * x[y][e].z; acc[e][3] += f * x[y][e].w;
        }
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    s_out[lane][4 * warp + 2 * e] = pack_bf16(acc[e][0] * inv, acc[e][1] * inv);
    s_out[lane][4 * warp + 2 * e + 1] = pack_bf16(acc[e][2] * inv, acc[e][3] * inv);
  }
  __syncthreads();
  // 64 bytes of a row: four threads
  const int row = threadIdx.x >> 2, piece = threadIdx.x & 3, q = rr0 + row;
  if (q >= rows) return;
  const int node = z * p.group_tokens + q / p.gqa, head = h * p.gqa + q % p.gqa;
  *reinterpret_cast<uint4*>(p.out + (r0 + node) * p.ldo + head * D + c0 + 8 * piece) =
      make_uint4(s_out[row][4 * piece], s_out[row][4 * piece + 1], s_out[row][4 * piece + 2], s_out[row][4 * piece + 3]);
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

// Places on the line of tiles are 32-bit numbers.
bool too_long(const B2TreeStep& t, int n_kv) { return (long long)t.requests * n_kv * (t.max_blocks / 4 + 2) >= 1ll << 30; }

// Query tiles of a CTA, nodes to a CTA, CTAs over the same keys, columns of CTAs.  The host knows what a step can hold, not what it holds, and a step
// made for more pays for it: 32 requests of 16 nodes, 40 heads on 8, in a step for trees of 16 / of 64 nodes 382 / 880 us (groups without rows, the second
// query tile empty), one request 18.0 / 20.2; one of 300 positions in a table of that / of 8192 positions 11.2 / 12.3.
struct Shape {
  int nw, tokens, groups, columns, single;
};
Shape shape_of(int B, int max_blocks, int n_kv, int gqa, int max_nodes) {
  Shape s;
  // One query tile on two groups in turn, or two query tiles.  64 nodes x 4 heads as 256 rows of one CTA / as 128 of
  // two CTAs over the same keys: 66 / 78 us; 16 nodes x 5 heads, 80 rows, with the second group idle: 394 -> 466, in 8 bits (24 x 5) 406 -> 608.
  s.nw = max_nodes * gqa <= BQ ? 1 : 2;
  const int most = s.nw * BQ / gqa;
  s.groups = (max_nodes + most - 1) / most;
  s.tokens = (max_nodes + s.groups - 1) / s.groups;
  // Short tables of few requests: a request's key head is one CTA's, and the second launch is spared.  Full tables, 32 heads on 8, one CTA / parts
  // that are added up, us: 1 request 9.7 / 10.4 at 6 tiles, 11.8 / 11.4 at 10; 16 requests 11.1 / 13.6 and 14.9 / 16.9; 32 requests (256 CTAs)
  // 22.6 / 28.0 and 29.4 / 33.9, at 18 39.9 / 43.2 and 1 request 15.7 / 15.4; 48 requests 28.9 / 25.5 at 3 tiles, 128 requests 82 / 62 at 6.
  // (A bound, not the best of both everywhere: 8 to 32 requests at 18 tiles lose 5 to 10 % by it, 1 request at 10 and 32 at 3 tiles 2 to 3 %.)
  const int most_tiles = max_blocks / 4 + 2;
  s.single = most_tiles <= 10 && (long long)B * n_kv * s.groups <= 2 * sm_count() ? most_tiles : 0;
  if (s.single) {
    s.columns = B * n_kv;
    return s;
  }
  const long long units = (long long)B * n_kv * most_tiles;      // tiles there can be
  const long long c = (long long)sm_count() / s.groups;
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
  if (rc || s.single) return rc;
  const int most = s.tokens * p.gqa;
  return b2_launch(tree_merge_kernel<F::D>, dim3((unsigned)(p.B * p.n_kv * s.groups), (unsigned)((most + 31) / 32 * (F::D / 32))), dim3(128), 0, st, true, p, s.columns,
                   s.nw * BQ, s.groups);
}

}  // namespace

// Tensor maps of a bf16 cache's first layer into the structure.
extern "C" int b2_tree_cache(B2TreeCache* c) {
  if (c->k_scale || (c->d != 64 && c->d != 128)) return c->k_scale ? 0 : -1;
  const uint64_t rows = (uint64_t)c->pages * c->heads * kPage;
  const int rc = cache_map(&c->map_k, c->k, rows, c->d);
  return rc ? rc : cache_map(&c->map_v, c->v, rows, c->d);
}

// fp32 words of workspace for b2_tree_attention on the current device
extern "C" long long b2_tree_attention_work(const B2TreeStep* t, int n_q, int n_kv, int D) {
  const Shape s = shape_of(t->requests, t->max_blocks, n_kv, n_q / n_kv, t->max_nodes);
  return (s.single ? 0 : 2ll * s.groups * s.columns * s.nw * BQ * (D + 2)) + (2 * t->requests + 2 + 3) / 4 * 4;
}

extern "C" int b2_tree_attention(const B2TreeStep* step, const B2TreeCache* cache, const void* q, long long ldq, void* out, long long ldo, float* work, int rows,
                                 int n_q, int window, float scale, void* stream) {
  const B2TreeStep& t = *step;
  const B2TreeCache& c = *cache;
  if (rows < 1 || t.requests < 1 || t.requests > kMaxReq || n_q < 1 || c.heads < 1 || n_q % c.heads || n_q / c.heads > 64 || (c.d != 64 && c.d != 128) || t.max_nodes < 1 ||
      t.max_nodes > kMaxNodes || c.pages < 1 || too_long(t, c.heads))
    return -1;
  if (((uintptr_t)q | (uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)out | (uintptr_t)work | (uintptr_t)c.k_scale | (uintptr_t)c.v_scale) % 16 || ldq % 8 || ldo % 8) return -2;
  const Shape s = shape_of(t.requests, t.max_blocks, c.heads, n_q / c.heads, t.max_nodes);
  TreeAttnParams p;
  p.q = (const __nv_bfloat16*)q; p.ldq = ldq; p.k8 = (const int8_t*)c.k; p.v8 = (const int8_t*)c.v; p.k_scale = c.k_scale; p.v_scale = c.v_scale;
  p.lengths = t.lengths; p.row_start = t.row_start; p.row_pos = t.row_pos; p.block_table = t.block_table; p.tree_table = t.tree_table;
  p.masks = t.masks; p.B = t.requests; p.max_blocks = t.max_blocks; p.tree_blocks = t.tree_blocks; p.num_pages = c.pages; p.rows = rows;
  p.n_q = n_q; p.n_kv = c.heads; p.gqa = n_q / c.heads; p.window = window; p.group_tokens = s.tokens; p.scale_log2 = scale * 1.4426950408889634f;
  p.out = (__nv_bfloat16*)out; p.ldo = ldo;
  const size_t slots = s.single ? 0 : 2ull * s.groups * s.columns * s.nw * BQ;
  p.single = s.single;
  p.part_o = work; p.part_ml = work + slots * c.d; p.sched = reinterpret_cast<int*>(work + slots * (c.d + 2));
  const CUtensorMap &mk = c.map_k, &mv = c.map_v;
  const cudaStream_t st = (cudaStream_t)stream;
  switch ((c.d == 128 ? 4 : 0) + (c.k_scale ? 2 : 0) + s.nw - 1) {
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
