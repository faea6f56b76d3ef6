// Attention of token trees over a paged cache: row i, a node of its request's tree, sees the request's cached positions and its own
// ancestors (bit j of its mask: node j), whose keys and values stand in the tree's pages.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j      j: cached positions < length, nodes of the mask; with a window those less than
//                                                   `window` positions before the row
//
// A row that sees nothing is 0.
#include "common.cuh"

using namespace b2;

namespace {

constexpr int kPage = 16;

struct TreeAttnParams {
  const __nv_bfloat16* q;
  long long ldq;
  const void *k, *v;
  const float *k_scale, *v_scale;
  const int *lengths, *row_start, *row_req, *row_pos, *block_table, *tree_table;
  const unsigned long long* masks;
  int B, max_blocks, tree_blocks, num_pages, max_rows, n_q, n_kv, window;
  float scale_log2;
  __nv_bfloat16* out;
  long long ldo;
};

// A CTA per row and head; its four warps take every fourth key and meet at the end.
template <int D, bool I8>
__global__ void __launch_bounds__(128) tree_attn_kernel(const TreeAttnParams p) {
  constexpr int E = D / 32;
  __shared__ float s_o[4][D], s_m[4], s_l[4];
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x, head = blockIdx.y, kh = head / (p.n_q / p.n_kv), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int req = p.row_req[row];
  if (req < 0 || req >= p.B) return;
  const int length = p.lengths[req], r0 = p.row_start[req], n = min(p.row_start[req + 1] - r0, 64);
  const unsigned long long mask = p.masks[row];
  const int lo = p.window > 0 ? p.row_pos[row] - p.window + 1 : 0;      // the first position that is seen
  float q[E], o[E], m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(p.q[row * p.ldq + head * D + lane * E + e]) * p.scale_log2;
    o[e] = 0.f;
  }
  for (int j = min(max(0, lo), length) + warp; j < length + n; j += 4) {
    int page, place;
    if (j < length) {
      page = j / kPage < p.max_blocks ? p.block_table[(size_t)req * p.max_blocks + j / kPage] : -1;
      place = j % kPage;
    } else {
      const int i = j - length;
      if (!(mask >> i & 1) || p.row_pos[r0 + i] < lo) continue;
      page = p.tree_table[(size_t)req * p.tree_blocks + i / kPage];
      place = i % kPage;
    }
    if (page < 0 || page >= p.num_pages) continue;
    const size_t at = ((size_t)page * p.n_kv + kh) * kPage + place;
    float s = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const size_t x = at * D + lane * E + e;
      s += q[e] * (I8 ? (float)((const int8_t*)p.k)[x] : __bfloat162float(((const __nv_bfloat16*)p.k)[x]));
      v[e] = I8 ? (float)((const int8_t*)p.v)[x] : __bfloat162float(((const __nv_bfloat16*)p.v)[x]);
    }
    s = warp_sum(s) * (I8 ? p.k_scale[at] : 1.f);
    const float mn = fmaxf(m, s), c = exp2f(m - mn), w = exp2f(s - mn), vs = I8 ? p.v_scale[at] : 1.f;
    m = mn;
    sum = sum * c + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * c + w * vs * v[e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = sum; }
  __syncthreads();
  const float best = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  for (int d = threadIdx.x; d < D; d += 128) {
    float total = 0.f, acc = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float c = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - best);
      total += c * s_l[w];
      acc += c * s_o[w][d];
    }
    p.out[row * p.ldo + head * D + d] = __float2bfloat16(total > 0.f ? acc / total : 0.f);
  }
}

}  // namespace

extern "C" int b2_tree_attention(const void* q, long long ldq, const void* k, const void* v, const float* k_scale, const float* v_scale, const int* lengths,
                                 const int* row_start, const int* row_req, const int* row_pos, const int* block_table, const int* tree_table,
                                 const void* masks, void* out, long long ldo, int rows, int B, int max_blocks, int tree_blocks, int num_pages, int n_q,
                                 int n_kv, int D, int window, float scale, void* stream) {
  if (rows < 1 || B < 1 || n_q < 1 || n_kv < 1 || n_q % n_kv || (D != 64 && D != 128)) return -1;
  TreeAttnParams p;
  p.q = (const __nv_bfloat16*)q; p.ldq = ldq; p.k = k; p.v = v; p.k_scale = k_scale; p.v_scale = v_scale; p.lengths = lengths; p.row_start = row_start;
  p.row_req = row_req; p.row_pos = row_pos; p.block_table = block_table; p.tree_table = tree_table; p.masks = (const unsigned long long*)masks;
  p.B = B; p.max_blocks = max_blocks; p.tree_blocks = tree_blocks; p.num_pages = num_pages; p.max_rows = rows; p.n_q = n_q; p.n_kv = n_kv;
  p.window = window; p.scale_log2 = scale * 1.4426950408889634f; p.out = (__nv_bfloat16*)out; p.ldo = ldo;
  const dim3 grid(rows, n_q);
  const auto kernel = D == 64 ? (k_scale ? tree_attn_kernel<64, true> : tree_attn_kernel<64, false>) : (k_scale ? tree_attn_kernel<128, true> : tree_attn_kernel<128, false>);
  return b2_launch(kernel, grid, dim3(128), 0, (cudaStream_t)stream, true, p);
}

B2_DEFINE_STATUS(treeattn)
