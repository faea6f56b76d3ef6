// Rotation of a step's rows and their way into the paged cache: row r of a qkv projection stands at position pos[r], its keys and values
// go to cache slot slot[r] (page x 16 + place), wherever that is.
//
//   y = x turned: pairs (i, i + n) or (2 i, 2 i + 1) of a head's first 2 n dimensions,  (a, b) -> (a cos - b sin, b cos + a sin)
//   q as bf16 rows; k and v as bf16, or as 8-bit integers with a scale per row and head, max|y| / 127 (1 where all are 0)
//
// Rows without a slot (-1) are left as they are.  Products and sums are rounded one by one, as the definition says them: an 8-bit value
// next to a border then is the same number whoever computes it.
//
// The bytes are the bound.  A thread takes four pairs of a head -- eight dimensions, in two pieces of four -- of HC heads of a row: a pair needs no
// other thread, and cosines and sines are read once for the row's heads.  All of a thread's loads are in flight together, and stay as they came
// until their turn.  5000 rows of 32 + 8 + 8 heads, bf16: 24.3 us (5.2 TB/s) with four heads a thread and five CTAs an SM; 26.0 with as many
// registers as it likes, 28.1 / 29.0 with two / eight heads; unpacked as they come 33 to 36, which leaves half the bytes under way.
// 16 rows, four slices: 2.1 us with a head a thread.  1008 rows of 16 + 4 + 4 heads into 8 bits: 7.4 us (18 MB, 2.8 us of bytes; what the rest is was not
// measured: heads of queries come by the scales' shuffles too, and 8-bit values leave four at a time).
#include "tree.cuh"

using namespace b2;

namespace {

constexpr int kPage = kTreePage;

struct TreeRopeParams {
  const void* qkv;          // bf16 [rows][ld], or fp32 [slices][rows][ld], slices added in order
  long long ld, slice;      // elements
  int slices;               // 0: bf16
  const int *pos, *slots;
  int rows;
  const float *cos_t, *sin_t;      // [positions][pairs]
  int pairs, positions, interleaved;
  int n_q, n_kv;
  __nv_bfloat16* q;
  long long ldq;
  void *k, *v;
  float *k_scale, *v_scale;        // null: bf16 cache
  long long num_slots;
  int chunks;                      // groups of HC heads in a row
};

template <int D, int HC, bool F32>
__global__ void __launch_bounds__(256, HC == 4 ? 5 : 1) tree_rope_kernel(const TreeRopeParams p) {
  constexpr int G = D / 8;             // threads to a head
  pdl_wait();
  pdl_launch_dependents();
  const int heads = p.n_q + 2 * p.n_kv, n_turn = p.n_q + p.n_kv;
  const int l = threadIdx.x % G, item = blockIdx.x * (256 / G) + threadIdx.x / G;
  const int row = min(item / p.chunks, p.rows - 1), h0 = (item - (item / p.chunks) * p.chunks) * HC;      // (groups past the end go along for the shuffles)
  const int pos = p.pos[row], slot = p.slots[row];
  bool live = item < p.rows * p.chunks && slot >= 0;
  if (live && (pos < 0 || pos >= p.positions || slot >= p.num_slots)) {
    if (l == 0) record_error(ERR_BAD_ARG, row);
    live = false;
  }
  // ---- the thread's dimensions: two pieces of four, off_a and off_b
  const bool turn = 4 * l < p.pairs;
  const int off_a = turn && !p.interleaved ? 4 * l : 8 * l, off_b = turn && !p.interleaved ? p.pairs + 4 * l : 8 * l + 4;
  // as they came until their turn: 16 (bf16) or 32 bytes a head on their way in few registers
  constexpr int NR = F32 ? 8 : 4;
  uint32_t raw[HC][NR];
#pragma unroll
  for (int c = 0; c < HC; ++c) {
    if (h0 + c >= heads) continue;      // (a row without a slot is read all the same: its number is not waited for)
    if constexpr (F32) {
      const float* src = reinterpret_cast<const float*>(p.qkv) + row * p.ld + (h0 + c) * D;
      *reinterpret_cast<uint4*>(raw[c]) = *reinterpret_cast<const uint4*>(src + off_a);
      *reinterpret_cast<uint4*>(raw[c] + 4) = *reinterpret_cast<const uint4*>(src + off_b);
    } else {
      const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(p.qkv) + row * p.ld + (h0 + c) * D;
      *reinterpret_cast<uint2*>(raw[c]) = *reinterpret_cast<const uint2*>(src + off_a);
      *reinterpret_cast<uint2*>(raw[c] + 2) = *reinterpret_cast<const uint2*>(src + off_b);
    }
  }
  float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live && turn && h0 < n_turn) {
    cs = __ldg(reinterpret_cast<const float4*>(p.cos_t + (size_t)pos * p.pairs) + l);
    sn = __ldg(reinterpret_cast<const float4*>(p.sin_t + (size_t)pos * p.pairs) + l);
  }
  const float cc[4] = {cs.x, cs.y, cs.z, cs.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
  for (int c = 0; c < HC; ++c) {
    const int head = h0 + c;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = head >= heads ? 0.f : F32 ? __uint_as_float(raw[c][e]) : e & 1 ? bf16_hi(raw[c][e >> 1]) : bf16_lo(raw[c][e >> 1]);
    if constexpr (F32) {
#pragma unroll 4
      for (int s = 1; s < p.slices; ++s) {
        if (head >= heads) continue;
        const float* src = reinterpret_cast<const float*>(p.qkv) + s * p.slice + row * p.ld + head * D;
        const float4 a = *reinterpret_cast<const float4*>(src + off_a), b = *reinterpret_cast<const float4*>(src + off_b);
        x[0] += a.x; x[1] += a.y; x[2] += a.z; x[3] += a.w; x[4] += b.x; x[5] += b.y; x[6] += b.z; x[7] += b.w;
      }
    }
    if (turn && head < n_turn) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = p.interleaved ? x[2 * e] : x[e], b = p.interleaved ? x[2 * e + 1] : x[4 + e];
        const float ya = __fsub_rn(__fmul_rn(a, cc[e]), __fmul_rn(b, ss[e])), yb = __fadd_rn(__fmul_rn(b, cc[e]), __fmul_rn(a, ss[e]));
        if (p.interleaved) { x[2 * e] = ya; x[2 * e + 1] = yb; } else { x[e] = ya; x[4 + e] = yb; }
      }
    }
    const bool is_q = head < p.n_q, is_v = head >= n_turn;
    const bool write = live && head < heads;
    __nv_bfloat16* dst = nullptr;
    long long at = 0;
    if (is_q) {
      dst = p.q + row * p.ldq + head * D;
    } else {
      at = ((long long)(max(slot, 0) / kPage) * p.n_kv + (head - (is_v ? n_turn : p.n_q))) * kPage + max(slot, 0) % kPage;
      dst = reinterpret_cast<__nv_bfloat16*>(is_v ? p.v : p.k) + at * D;
    }
    if (is_q || !p.k_scale) {
      if (write) {
        *reinterpret_cast<uint2*>(dst + off_a) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
        *reinterpret_cast<uint2*>(dst + off_b) = make_uint2(pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
      }
    }
    if (p.k_scale) {
      float largest = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(x[e]));
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o, G));
      if (write && !is_q) {
        const float scale = largest > 0.f ? largest / 127.f : 1.f, inv = 1.f / scale;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2] |= (uint32_t)(__float2int_rn(__fmul_rn(x[e], inv)) & 0xff) << (8 * (e & 3));
        int8_t* d8 = reinterpret_cast<int8_t*>(is_v ? p.v : p.k) + at * D;
        *reinterpret_cast<uint32_t*>(d8 + off_a) = w[0];
        *reinterpret_cast<uint32_t*>(d8 + off_b) = w[1];
        if (l == 0) (is_v ? p.v_scale : p.k_scale)[at] = scale;
      }
    }
  }
}

template <int D, bool F32>
int launch(const TreeRopeParams& q, cudaStream_t st) {
  TreeRopeParams p = q;
  const int heads = p.n_q + 2 * p.n_kv;
  const long long items = (long long)p.rows * heads;
  // Four heads a thread where that still gives every SM 2048 threads; below, a head each: more threads, shorter ways.
  const bool four = items * (D / 8) >= 4ll * 148 * 2048;
  p.chunks = four ? (heads + 3) / 4 : heads;
  const long long groups = (long long)p.rows * p.chunks, per = 256 / (D / 8);
  if (groups > 0x7fffffffll - 1024) return -3;
  const dim3 grid((unsigned)((groups + per - 1) / per));
  if (four) return b2_launch(tree_rope_kernel<D, 4, F32>, grid, dim3(256), 0, st, true, p);
  return b2_launch(tree_rope_kernel<D, 1, F32>, grid, dim3(256), 0, st, true, p);
}

}  // namespace

extern "C" int b2_tree_rope(const B2TreeStep* step, const B2TreeCache* cache, const void* qkv, long long ld, long long slice, int slices, int rows, const float* cos_t,
                            const float* sin_t, int pairs, int positions, int interleaved, int n_q, void* q, long long ldq, void* stream) {
  const B2TreeCache& c = *cache;
  if (rows < 1 || rows > step->max_rows || (c.d != 64 && c.d != 128) || pairs < 0 || pairs % 4 || 2 * pairs > c.d || n_q < 1 || c.heads < 1) return -1;
  if (((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)cos_t | (uintptr_t)sin_t) % 16 || ld % 4 || ldq % 4 || slice % 4) return -2;
  TreeRopeParams p;
  p.qkv = qkv; p.ld = ld; p.slice = slice; p.slices = slices; p.pos = step->row_pos; p.slots = step->slots; p.rows = rows; p.cos_t = cos_t; p.sin_t = sin_t;
  p.pairs = pairs; p.positions = positions; p.interleaved = interleaved; p.n_q = n_q; p.n_kv = c.heads; p.q = (__nv_bfloat16*)q; p.ldq = ldq;
  p.k = c.k; p.v = c.v; p.k_scale = c.k_scale; p.v_scale = c.v_scale; p.num_slots = (long long)c.pages * kPage; p.chunks = 0;
  const cudaStream_t st = (cudaStream_t)stream;
  if (c.d == 64) return slices ? launch<64, true>(p, st) : launch<64, false>(p, st);
  return slices ? launch<128, true>(p, st) : launch<128, false>(p, st);
}

B2_DEFINE_STATUS(treerope)
