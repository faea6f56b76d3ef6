// Rotation of a step's rows and their way into the paged cache: row r of a qkv projection stands at position pos[r], its keys and values
// go to cache slot slot[r] (page x 16 + place), wherever that is.
//
//   y = x turned: pairs (i, i + n) or (2 i, 2 i + 1) of a head's first 2 n dimensions,  (a, b) -> (a cos - b sin, b cos + a sin)
//   q as bf16 rows; k and v as bf16, or as 8-bit integers with a scale per row and head, max|y| / 127 (1 where all are 0)
//
// Rows without a slot (-1) are left as they are.  Products and sums are rounded one by one, as the definition says them: an 8-bit value
// next to a border then is the same number whoever computes it.
#include "common.cuh"

using namespace b2;

namespace {

constexpr int kPage = 16;

struct TreeRopeParams {
  const void* qkv;          // bf16 [rows][ld], or fp32 [slices][rows][ld], slices added in order
  long long ld, slice;      // elements
  int slices;               // 0: bf16
  const int *pos, *slots;
  int rows;
  const float *cos_t, *sin_t;      // [positions][rot / 2]
  int rot, positions, interleaved;
  int n_q, n_kv, D;
  __nv_bfloat16* q;
  long long ldq;
  void *k, *v;
  float *k_scale, *v_scale;        // null: bf16 cache
  long long num_slots;
};

// D / 4 lanes take a row's head, four dimensions each.
template <int D>
__global__ void __launch_bounds__(256) tree_rope_kernel(const TreeRopeParams p) {
  constexpr int G = D / 4;
  pdl_wait();
  pdl_launch_dependents();
  const int heads = p.n_q + 2 * p.n_kv;
  const int l = threadIdx.x % G, item = blockIdx.x * (256 / G) + threadIdx.x / G;
  const int row = min(item / heads, p.rows - 1), head = item - (item / heads) * heads;      // (groups past the end go along for the shuffles)
  const int pos = p.pos[row], slot = p.slots[row];
  bool live = item < p.rows * heads && slot >= 0;
  if (live && (pos < 0 || pos >= p.positions || slot >= p.num_slots)) {
    if (l == 0) record_error(ERR_BAD_ARG, row);
    live = false;
  }
  const int e = head * D + 4 * l;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    if (p.slices) {
      const float* src = reinterpret_cast<const float*>(p.qkv) + row * p.ld + e;
      float4 a = *reinterpret_cast<const float4*>(src);
#pragma unroll 4
      for (int s = 1; s < p.slices; ++s) {
        const float4 t = *reinterpret_cast<const float4*>(src + s * p.slice);
        a.x += t.x; a.y += t.y; a.z += t.z; a.w += t.w;
      }
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    } else {
      const uint2 t = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(p.qkv) + row * p.ld + e);
      x[0] = bf16_lo(t.x); x[1] = bf16_hi(t.x); x[2] = bf16_lo(t.y); x[3] = bf16_hi(t.y);
    }
  }
  if (head < p.n_q + p.n_kv || !live) {      // (lanes of one head go the same way; dead ones come along)
    const int half = p.rot >> 1;
    if (p.interleaved) {
      if (live && 4 * l < p.rot) {
        const float2 c = *reinterpret_cast<const float2*>(p.cos_t + (size_t)pos * half + 2 * l), s = *reinterpret_cast<const float2*>(p.sin_t + (size_t)pos * half + 2 * l);
        const float a0 = x[0], b0 = x[1], a1 = x[2], b1 = x[3];
        x[0] = __fsub_rn(__fmul_rn(a0, c.x), __fmul_rn(b0, s.x));
        x[1] = __fadd_rn(__fmul_rn(b0, c.x), __fmul_rn(a0, s.x));
        x[2] = __fsub_rn(__fmul_rn(a1, c.y), __fmul_rn(b1, s.y));
        x[3] = __fadd_rn(__fmul_rn(b1, c.y), __fmul_rn(a1, s.y));
      }
    }
  }
  {
    const int half = p.rot >> 1, hl = half >> 2;       // lanes of half the rotated part
    const bool low = l < hl;
    const int other = low ? l + hl : l - hl;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], other & (G - 1), G);
    if (!p.interleaved && live && head < p.n_q + p.n_kv && l < 2 * hl) {
      const int j = 4 * (low ? l : l - hl);
      const float4 c = *reinterpret_cast<const float4*>(p.cos_t + (size_t)pos * half + j), s = *reinterpret_cast<const float4*>(p.sin_t + (size_t)pos * half + j);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] = low ? __fsub_rn(__fmul_rn(x[i], cc[i]), __fmul_rn(y[i], ss[i])) : __fadd_rn(__fmul_rn(x[i], cc[i]), __fmul_rn(y[i], ss[i]));
    }
  }
  if (head < p.n_q) {
    if (live) *reinterpret_cast<uint2*>(p.q + row * p.ldq + e) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
    if (!p.k_scale) return;
  }
  const bool is_v = head >= p.n_q + p.n_kv;
  const int kh = is_v ? head - p.n_q - p.n_kv : head - p.n_q;
  const long long at = live && head >= p.n_q ? ((long long)(slot / kPage) * p.n_kv + kh) * kPage + slot % kPage : 0;
  if (!p.k_scale) {
    if (live) *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(is_v ? p.v : p.k) + at * D + 4 * l) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
    return;
  }
  float largest = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o, G));
  if (!live || head < p.n_q) return;
  const float scale = largest > 0.f ? largest / 127.f : 1.f, inv = 1.f / scale;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= (uint32_t)(__float2int_rn(__fmul_rn(x[i], inv)) & 0xff) << (8 * i);
  *reinterpret_cast<uint32_t*>(reinterpret_cast<int8_t*>(is_v ? p.v : p.k) + at * D + 4 * l) = w;
  if (l == 0) (is_v ? p.v_scale : p.k_scale)[at] = scale;
}

}  // namespace

extern "C" int b2_tree_rope(const void* qkv, long long ld, long long slice, int slices, const int* pos, const int* slots, int rows, const float* cos_t,
                            const float* sin_t, int rot, int positions, int interleaved, int n_q, int n_kv, int D, void* q, long long ldq, void* k,
                            void* v, float* k_scale, float* v_scale, long long num_slots, void* stream) {
  if (rows < 1 || (D != 64 && D != 128) || rot < 0 || rot % 8 || rot > D || n_q < 1 || n_kv < 1) return -1;
  if (((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cos_t | (uintptr_t)sin_t) % 16 || ld % 4 || ldq % 4 || slice % 4) return -2;
  TreeRopeParams p;
  p.qkv = qkv; p.ld = ld; p.slice = slice; p.slices = slices; p.pos = pos; p.slots = slots; p.rows = rows; p.cos_t = cos_t; p.sin_t = sin_t;
  p.rot = rot; p.positions = positions; p.interleaved = interleaved; p.n_q = n_q; p.n_kv = n_kv; p.D = D; p.q = (__nv_bfloat16*)q; p.ldq = ldq;
  p.k = k; p.v = v; p.k_scale = k_scale; p.v_scale = v_scale; p.num_slots = num_slots;
  const long long items = (long long)rows * (n_q + 2 * n_kv), per = 256 / (D / 4);
  if (items > 0x7fffffffll - 1024) return -3;
  const dim3 grid((unsigned)((items + per - 1) / per));
  if (D == 64) return b2_launch(tree_rope_kernel<64>, grid, dim3(256), 0, (cudaStream_t)stream, true, p);
  return b2_launch(tree_rope_kernel<128>, grid, dim3(256), 0, (cudaStream_t)stream, true, p);
}

B2_DEFINE_STATUS(treerope)
