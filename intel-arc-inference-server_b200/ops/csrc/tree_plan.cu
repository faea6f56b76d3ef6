// Steps over token trees: what a step's rows are and where they stand (plan), and what stays of them (commit).
//
//   plan    lengths, rows and pages of every request -> first rows, and of every row its request, position, cache slot, parent and
//           ancestors; new pages come off the end of a free list into the block table
//   commit  the accepted path of every tree (node 0, then the child whose token is its parent's target, as long as there is one); the
//           path's keys and values move from the tree's pages to the request's positions, in all layers
//
// Plan is one CTA, or one cluster of eight: everything hangs on three prefix sums over the requests, and with the few pages that a step takes a launch is
// all that a call costs.  (A request's pages are one thread's, one after another: a first prompt of 33000 positions 75 us, a request of 131072 that leaves
// 1.3 ms.)  Device time in a row of calls: one tree of 16 nodes 4.2 us (5.3 with parents read from memory at every step up), 100 requests with 8050 rows 6.4 (one CTA:
// 11.4); their 0.2 MB are 0.03 us of bytes.
#include "tree.cuh"

using namespace b2;

namespace {

constexpr int kPage = kTreePage, kMaxNodes = kTreeNodes, kMaxReq = kTreeRequests;
constexpr int kUpRows = 8192;      // rows whose parents are kept in shared memory

enum : int { PLAN_POOL = 1, PLAN_TABLE = 2, PLAN_ROWS = 4, PLAN_COUNT = 8, PLAN_PARENT = 16, PLAN_LENGTH = 32, PLAN_PAGE = 64 };

struct TreePlanParams {
  const int *lengths, *counts, *parents;   // parents null: rows at consecutive positions
  int* block_table;
  const int* tree_table;
  int* free;
  const int *n_free, *held;
  int *n_free_out, *held_out;
  int B, max_blocks, tree_blocks, free_cap, max_rows, max_nodes, num_pages;
  int rows;                                // parents there are (max_rows without)
  int *out_lengths, *row_start, *row_req, *row_pos, *slots, *out_parents, *status;
  unsigned long long* masks;
};

// Exclusive prefix sums of one number per thread over the CTA; the total in `total`.
template <typename T>
__device__ __forceinline__ T scan_cta(T v, long long* warp_sums, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  T x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  T w = lane < warps ? (T)warp_sums[lane] : 0;      // every warp for itself
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const T before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return x - v + (warp ? before : 0);
}

__device__ __forceinline__ int cluster_rank() { int r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ int cluster_size() { int r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A cluster of one CTA, or of eight where there are more rows than one CTA's threads: each does the sums for itself (there is nothing to wait for
// that way), the first one keeps the pages, all of them write rows.  A request a thread.
// What is at fault with the numbers, the trees, the pages and the rows are four words: each is written up to a barrier that is everyone's and only
// looked at behind it, since what threads go by must not change while others still look.
__global__ void __launch_bounds__(1024, 1) tree_plan_kernel(const TreePlanParams p) {
  __shared__ long long sums[32];
  __shared__ int s_start[kMaxReq + 1], s_need[kMaxReq], s_held[kMaxReq], s_first[kMaxReq], s_len[kMaxReq];
  __shared__ int8_t s_up[kUpRows];
  __shared__ int s_numbers, s_trees, s_pages, s_rows;
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, rank = cluster_rank(), ranks = cluster_size();
  pdl_wait();
  pdl_launch_dependents();
  const bool tree = p.parents != nullptr, mine = tid < p.B, up_here = tree && p.rows <= kUpRows;
  if (tid == 0) s_numbers = s_trees = s_pages = s_rows = 0;
  const int count = mine ? p.counts[tid] : 0, held = mine ? p.held[tid] : 0, n_free = *p.n_free;
  const int given = mine ? p.lengths[tid] : 0, length = count >= 0 ? given : 0;
  if (up_here)
    for (int r = tid; r < p.rows; r += threads) {
      const int up = p.parents[r];
      s_up[r] = up >= -1 && up < kMaxNodes ? (int8_t)up : (int8_t)127;      // (127: before no node)
    }
  auto parent = [&](int r) { return up_here ? (int)s_up[r] : p.parents[r]; };
  __syncthreads();
  if (mine) {
    int bad = 0;
    if (length < 0) bad |= PLAN_LENGTH;
    if (held < 0 || held > p.max_blocks) bad |= PLAN_TABLE;
    if (tree && count > p.max_nodes) bad |= PLAN_COUNT;
    if (n_free < 0 || n_free > p.free_cap) bad |= PLAN_POOL;
    if (bad) atomicOr(&s_numbers, bad);
  }
  int total;
  const int start = scan_cta(min(max(count, 0), p.rows + 1), sums, total);      // (at most 2^20 + 1 each)
  if (total > p.rows && tid == 0) atomicOr(&s_numbers, PLAN_ROWS);
  if (mine) {
    s_start[tid] = min(start, p.rows);
    s_need[tid] = tree ? 0 : max(count, 0);
    s_held[tid] = held;
    s_len[tid] = length;
  }
  if (tid == 0) s_start[p.B] = min(total, p.rows);
  __syncthreads();
  if (s_numbers == 0 && tree) {
    // ---- a warp per tree: ancestors by walking up (a node's parent stands before it, so every walk ends)
    for (int b = warp; b < p.B; b += threads >> 5) {
      const int r0 = s_start[b], n = s_start[b + 1] - r0;
      int deepest = 0;
      bool bad = false;
      for (int i = lane; i < n; i += 32) {
        const int up = parent(r0 + i);
        bad |= up < -1 || up >= i;
      }
      bad = __any_sync(0xffffffffu, bad);
      if (bad) {
        if (lane == 0) s_trees = PLAN_PARENT;
        continue;
      }
      for (int i = lane; i < n; i += 32) {
        int depth = 0;
        for (int at = i; at >= 0; at = parent(r0 + at)) ++depth;
        deepest = max(deepest, depth);
      }
      deepest = __reduce_max_sync(0xffffffffu, deepest);
      if (lane == 0) s_need[b] = deepest;
    }
  }
  __syncthreads();
  // ---- pages: those of requests that left go back, then what is missing comes off the end of the list
  const int need = mine && (s_numbers | s_trees) == 0 ? s_need[tid] : 0;
  const long long want = need > 0 ? max((long long)held, ((long long)length + need + kPage - 1) / kPage) : held;
  const bool left = mine && count < 0;
  if (mine && !left && want > p.max_blocks) atomicOr(&s_pages, PLAN_TABLE);
  long long back, take;
  const long long back0 = scan_cta(left ? (long long)held : 0ll, sums, back);
  const long long take0 = scan_cta(mine && !left ? want - held : 0ll, sums, take);
  if (mine) s_first[tid] = (int)take0;
  if (tid == 0 && ((long long)n_free + back > p.free_cap || take > (long long)n_free + back)) atomicOr(&s_pages, PLAN_POOL);
  __syncthreads();
  const int status = s_numbers | s_trees | s_pages;
  if (rank == 0 && tid == 0) p.status[0] = status;
  if (ranks > 1) cluster_barrier();      // everyone has read what the first CTA now writes
  const long long top = (long long)n_free + back - 1;     // the page that is taken first
  if (rank == 0 && status == 0 && left)
    for (int i = 0; i < held; ++i) {
      int* at = p.block_table + (size_t)tid * p.max_blocks + i;
      p.free[n_free + back0 + i] = *at;
      *at = 0;
    }
  if (back > 0) {      // pages that came back may be taken at once
    if (ranks > 1) cluster_barrier();
    else __syncthreads();
  }
  if (rank == 0) {
    if (status == 0 && mine && !left)
      for (int i = 0; i < (int)(want - held); ++i) p.block_table[(size_t)tid * p.max_blocks + held + i] = p.free[top - take0 - i];
    if (mine) {
      p.held_out[tid] = status ? held : left ? 0 : (int)want;
      p.out_lengths[tid] = status ? given : length;
    }
    if (tid == 0) p.n_free_out[0] = status ? n_free : (int)(n_free + back - take);
    for (int b = tid; b <= p.B; b += threads) p.row_start[b] = status ? 0 : s_start[b];
  }
  // ---- rows
  const int rows = status ? 0 : s_start[p.B];
  for (int r = rank * threads + tid; r < p.max_rows; r += ranks * threads) {
    int req = -1, pos = -1, slot = -1, up = -1;
    unsigned long long mask = 0;
    if (r < rows) {
      int lo = 0, hi = p.B - 1;       // the last request that starts at or before r
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_start[mid] <= r) lo = mid; else hi = mid - 1;
      }
      req = lo;
      const int i = r - s_start[req];
      int page;
      if (tree) {
        page = p.tree_table[(size_t)req * p.tree_blocks + i / kPage];
        up = parent(r);
        for (int at = i; at >= 0; at = parent(s_start[req] + at)) mask |= 1ull << at;
        pos = s_len[req] + __popcll(mask) - 1;
        slot = i % kPage;
      } else {
        pos = s_len[req] + i;
        const int block = pos / kPage;
        page = block < s_held[req] ? p.block_table[(size_t)req * p.max_blocks + block] : p.free[top - s_first[req] - (block - s_held[req])];
        slot = pos % kPage;
      }
      if (page < 0 || page >= p.num_pages) {
        s_rows = PLAN_PAGE;
        slot = -1;
      } else {
        slot += page * kPage;
      }
    }
    p.row_req[r] = req;
    p.row_pos[r] = pos;
    p.slots[r] = slot;
    if (tree) {
      p.masks[r] = mask;
      p.out_parents[r] = up;
    }
  }
  __syncthreads();
  if (tid == 0 && s_rows) atomicOr(p.status, s_rows);      // pages that are not there
}

struct TreeCommitParams {
  const int *lengths, *row_start, *parents, *tokens, *targets, *block_table, *tree_table;
  int B, max_blocks, tree_blocks, planes, num_pages, n_kv, rows;
  uint8_t *k, *v;
  long long plane_bytes;          // from plane to plane of k and v
  float *k_scale, *v_scale;
  long long plane_scales;
  int row_bytes;
  int *path, *count, *next_token, *out_lengths;
};

// A CTA per request and layer; each walks the tree for itself, a node or two to a lane, a child found by a vote (no second launch, nothing to wait for).
// Bound by its launch and four ways to memory one after another: one tree over 64 layers 3 to 4 us, 32 trees over 40 layers of 8 bits 6.5 to 8.2 (1.2 of bytes).
__global__ void __launch_bounds__(256) tree_commit_kernel(const TreeCommitParams p) {
  __shared__ int s_n, s_src[kMaxNodes], s_dst[kMaxNodes], s_path[kMaxNodes];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  pdl_wait();
  pdl_launch_dependents();
  if (tid < 32) {
    const int r0 = p.row_start[b], end = p.row_start[b + 1], length = p.lengths[b];
    const int n = min(end, p.rows) - r0;       // (fewer tokens than rows: an error below)
    if (end > p.rows && lane == 0 && blockIdx.y == 0) record_error(ERR_BAD_ARG, b);
    int at = 0, len = 0, next = -1;
    if (n > 0) {
      const int i0 = lane, i1 = lane + 32;
      const int up0 = i0 < n ? p.parents[r0 + i0] : -2, up1 = i1 < n ? p.parents[r0 + i1] : -2;
      const int tok0 = i0 < n ? p.tokens[r0 + i0] : 0, tok1 = i1 < n ? p.tokens[r0 + i1] : 0;
      const int tgt0 = i0 < n ? p.targets[r0 + i0] : 0, tgt1 = i1 < n ? p.targets[r0 + i1] : 0;
      for (;;) {
        if (lane == 0) s_path[len] = at;
        ++len;
        const int want0 = __shfl_sync(0xffffffffu, tgt0, at & 31), want1 = __shfl_sync(0xffffffffu, tgt1, at & 31);
        next = at < 32 ? want0 : want1;
        const unsigned f0 = __ballot_sync(0xffffffffu, up0 == at && tok0 == next && i0 > at);
        const unsigned f1 = __ballot_sync(0xffffffffu, up1 == at && tok1 == next && i1 > at);
        if (!(f0 | f1)) break;
        at = f0 ? __ffs(f0) - 1 : 31 + __ffs(f1);      // a child stands behind its parent: the walk ends
      }
    }
    __syncwarp();
    for (int i = lane; i < kMaxNodes; i += 32) {
      const int node = i < len ? s_path[i] : -1;
      if (i < len) {
        const int block = (length + i) / kPage;
        int src = p.tree_table[(size_t)b * p.tree_blocks + node / kPage], dst = block < p.max_blocks ? p.block_table[(size_t)b * p.max_blocks + block] : -1;
        if (src < 0 || src >= p.num_pages || dst < 0 || dst >= p.num_pages) {
          if (blockIdx.y == 0) record_error(ERR_BAD_ARG, b);
          src = dst = -1;
        }
        s_src[i] = src < 0 ? -1 : src * kPage * p.n_kv + node % kPage;
        s_dst[i] = src < 0 ? -1 : dst * kPage * p.n_kv + (length + i) % kPage;
      }
      if (blockIdx.y == 0) p.path[b * kMaxNodes + i] = node;
    }
    if (lane == 0) {
      s_n = len;
      if (blockIdx.y == 0) {
        p.count[b] = len;
        p.next_token[b] = next;
        p.out_lengths[b] = length + len;
      }
    }
  }
  __syncthreads();
  const int n = s_n, per = p.row_bytes >> 4, each = n * p.n_kv * per;
  for (int plane = blockIdx.y; plane < p.planes; plane += gridDim.y) {
    for (int j = tid; j < 2 * each; j += 256) {
      const int w = j >= each, e = w ? j - each : j;
      const int i = e / (p.n_kv * per), rest = e - i * p.n_kv * per, h = rest / per, piece = rest - h * per;
      if (s_src[i] < 0) continue;
      uint8_t* base = (w ? p.v : p.k) + plane * p.plane_bytes + 16 * piece;
      *reinterpret_cast<uint4*>(base + ((long long)s_dst[i] + h * kPage) * p.row_bytes) =
          *reinterpret_cast<const uint4*>(base + ((long long)s_src[i] + h * kPage) * p.row_bytes);
    }
    if (p.k_scale)
      for (int j = tid; j < 2 * n * p.n_kv; j += 256) {
        const int w = j >= n * p.n_kv, e = w ? j - n * p.n_kv : j, i = e / p.n_kv, h = e - i * p.n_kv;
        if (s_src[i] < 0) continue;
        float* base = (w ? p.v_scale : p.k_scale) + plane * p.plane_scales;
        base[(long long)s_dst[i] + h * kPage] = base[(long long)s_src[i] + h * kPage];
      }
  }
}

}  // namespace

// parents: of `rows` rows, or null (rows: the step's room)
extern "C" int b2_tree_plan(const B2TreeStep* step, const B2TreePool* pool, const B2TreePool* after, const int* lengths, const int* counts, const int* parents,
                            int rows, void* stream) {
  const B2TreeStep& t = *step;
  if (t.requests < 1 || t.requests > kMaxReq || rows < 0 || rows > t.max_rows || t.max_nodes < 1 || t.max_nodes > kMaxNodes || t.max_nodes > t.tree_blocks * kPage) return -1;
  TreePlanParams p;
  p.lengths = lengths; p.counts = counts; p.parents = parents; p.block_table = t.block_table; p.tree_table = t.tree_table; p.free = pool->free;
  p.n_free = pool->n_free; p.held = pool->held; p.n_free_out = after->n_free; p.held_out = after->held; p.out_lengths = t.lengths; p.row_start = t.row_start;
  p.row_req = t.row_req; p.row_pos = t.row_pos; p.slots = t.slots; p.out_parents = t.parents; p.masks = t.masks; p.status = t.status;
  p.B = t.requests; p.max_blocks = t.max_blocks; p.tree_blocks = t.tree_blocks; p.free_cap = pool->capacity; p.max_rows = t.max_rows; p.max_nodes = t.max_nodes;
  p.num_pages = t.num_pages; p.rows = rows;
  const int threads = t.requests <= 256 && t.max_rows <= 512 ? 256 : 1024, ctas = t.max_rows > 1024 ? 8 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = b2_no_pdl() ? 1 : 2;
  return (int)cudaLaunchKernelEx(&cfg, tree_plan_kernel, p);
}

// -3: results that overlap what is read (a request's CTAs, one per layer, each read everything, and one of them writes the results), or the step's other numbers
extern "C" int b2_tree_commit(const B2TreeStep* step, const B2TreeCache* cache, const B2TreeAccepted* accepted, const int* tokens, const int* targets, int rows,
                              void* stream) {
  const B2TreeStep& t = *step;
  const B2TreeCache& c = *cache;
  const int row_bytes = c.d * (c.k_scale ? 1 : 2);
  if (t.requests < 1 || t.requests > kMaxReq || c.layers < 1 || row_bytes % 16 || ((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.layer_bytes) % 16) return -1;
  const auto meet = [](const void* a, long long na, const void* b, long long nb) {
    return (uintptr_t)a < (uintptr_t)b + 4 * nb && (uintptr_t)b < (uintptr_t)a + 4 * na;
  };
  const long long B = t.requests;
  const struct { const void* at; long long n; } read[] = {{tokens, rows}, {targets, rows}, {t.lengths, B}, {t.row_start, B + 1}, {t.parents, t.max_rows},
                                                          {t.block_table, B * t.max_blocks}, {t.tree_table, B * t.tree_blocks}, {t.row_req, t.max_rows},
                                                          {t.row_pos, t.max_rows}, {t.slots, t.max_rows}, {t.masks, 2ll * t.max_rows}, {t.status, 1}};
  for (const auto& r : read)
    if (meet(r.at, r.n, accepted->path, B * kMaxNodes) || meet(r.at, r.n, accepted->count, B) || meet(r.at, r.n, accepted->next_token, B) ||
        meet(r.at, r.n, accepted->lengths, B))
      return -3;
  TreeCommitParams p;
  p.lengths = t.lengths; p.row_start = t.row_start; p.parents = t.parents; p.tokens = tokens; p.targets = targets; p.block_table = t.block_table;
  p.tree_table = t.tree_table; p.B = t.requests; p.max_blocks = t.max_blocks; p.tree_blocks = t.tree_blocks; p.planes = c.layers; p.num_pages = c.pages;
  p.n_kv = c.heads; p.rows = rows; p.k = (uint8_t*)c.k; p.v = (uint8_t*)c.v; p.plane_bytes = c.layer_bytes; p.k_scale = c.k_scale; p.v_scale = c.v_scale;
  p.plane_scales = c.layer_scales; p.row_bytes = row_bytes; p.path = accepted->path; p.count = accepted->count; p.next_token = accepted->next_token;
  p.out_lengths = accepted->lengths;
  return b2_launch(tree_commit_kernel, dim3(t.requests, min(c.layers, 65535)), dim3(256), 0, (cudaStream_t)stream, true, p);
}

B2_DEFINE_STATUS(tree)
