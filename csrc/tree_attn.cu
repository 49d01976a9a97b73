// Attention of drafted-token trees over the paged cache on the CUDA cores: every type, head width and page size that the tensor-core
// kernel (tree_attn_sm100.cu) does not take. Node i of tree b stands at cache position context[b] + i and sees the positions in front
// of context[b], the nodes above it and itself:
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(scale q_i k_j) / (sum_j' exp(scale q_i k_j') + exp(sink))
//
// One warp per (node, query head), 32 keys a turn: a lane works out the whole product of its key, the maximum and the sum of the softmax
// run along in fp32, then the lanes share the channels of the 32 values. A value with weight 0 is not read, so what stands in
// hidden or unwritten cache rows never reaches a sum. What bounds it is the latency of the lanes' key rows.
// The order of the sums is the same for every batch.
#include "token_tree.cuh"

namespace sb {

constexpr int TA_MAXD = 256;

template <typename T>
__global__ void __launch_bounds__(128)
tree_attn_kernel(const T* __restrict__ q, const T* __restrict__ k_cache, const T* __restrict__ v_cache, const int* __restrict__ table,
                 const int* __restrict__ context, const int* __restrict__ cu, const int* __restrict__ parents,
                 const float* __restrict__ sinks, T* __restrict__ out, int B, int Hq, int Hkv, int D, int page_size, int max_pages,
                 int num_slots, int max_nodes, long q_row, long q_head, long k_row, long k_head, long v_row, long v_head, long out_row,
                 float scale) {
  __shared__ float q_s[4][TA_MAXD];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x, h = blockIdx.y * 4 + warp;
  if (h >= Hq || t < cu[0] || t >= cu[B]) return;
  const int b = tree_of_row(cu, B, t);
  if (cu[b] < 0) return;
  const int i = t - cu[b], n = min(cu[b + 1] - cu[b], max_nodes);
  if (i >= n) return;
  const int kvh = h / (Hq / Hkv);
  const int ctx = min(max(context[b], 0), max_pages * page_size);
  const int total = min(ctx + n, max_pages * page_size);
  uint32_t above[4];
  const int* mine = parents + cu[b];
  tree_way_up([&](int j) { return mine[j]; }, i, above);
  const bool hole = (above[0] & 1) == 0;
  for (int d = lane; d < D; d += 32) q_s[warp][d] = static_cast<float>(q[t * q_row + h * q_head + d]);
  __syncwarp();
  const float c = scale * 1.4426950408889634f;
  float m = -INFINITY, l = 0.f, acc[TA_MAXD / 32];
#pragma unroll
  for (int x = 0; x < TA_MAXD / 32; ++x) acc[x] = 0.f;
  for (int k0 = 0; k0 < (hole ? 0 : total); k0 += 32) {
    const int key = k0 + lane, behind = key - ctx;
    bool sees = key < total;
    if (behind >= 0) {
      uint32_t word = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (behind >> 5 == w) word = above[w];
      sees = sees && (word >> (behind & 31) & 1);
    }
    long slot = 0;
    if (sees) {
      slot = static_cast<long>(table[static_cast<long>(b) * max_pages + key / page_size]) * page_size + key % page_size;
      sees = slot >= 0 && slot < num_slots;
    }
    float s = -INFINITY;
    if (sees) {
      const T* row = k_cache + slot * k_row + kvh * k_head;
      s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(q_s[warp][d], static_cast<float>(row[d]), s);
      s *= c;
    }
    if (!__any_sync(0xffffffffu, sees)) continue;
    const float top = fmaxf(m, warp_max(s)), zero = top == -INFINITY ? 0.f : top;  // (maxima leave NaN out, the weights below do not)
    const float keep = exp2f(m - zero), p = exp2f(s - zero);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int x = 0; x < TA_MAXD / 32; ++x) acc[x] *= keep;
    for (int j = 0; j < 32; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
      const long sj = __shfl_sync(0xffffffffu, slot, j);
      if (pj == 0.f) continue;
      const T* row = v_cache + sj * v_row + kvh * v_head;
#pragma unroll
      for (int x = 0; x < TA_MAXD / 32; ++x)
        if (x * 32 + lane < D) acc[x] = fmaf(pj, static_cast<float>(row[x * 32 + lane]), acc[x]);
    }
  }
  l = warp_sum(l);
  if (sinks != nullptr && m != -INFINITY) l += exp2f(sinks[h] * 1.4426950408889634f - m);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int x = 0; x < TA_MAXD / 32; ++x)
    if (x * 32 + lane < D) out[t * out_row + static_cast<long>(h) * D + x * 32 + lane] = static_cast<T>(acc[x] * inv);
}

}  // namespace sb

// q: rows of pitch q_row, heads of pitch q_head; caches: slots of pitch k_row / v_row, heads of pitch k_head / v_head; out: rows of pitch
// out_row, heads side by side (all in elements, channels adjacent). rows: packed rows of q and out. Rows behind cu[B] and beyond
// max_nodes of a tree are left as they are. Returns 0, a cudaError_t value, or -1 for heads wider than 256.
extern "C" int sb_tree_attn(const void* q, const void* k_cache, const void* v_cache, const int* table, const int* context, const int* cu,
                            const int* parents, const float* sinks, void* out, int rows, int B, int Hq, int Hkv, int D, int page_size,
                            int max_pages, int num_slots, int max_nodes, long q_row, long q_head, long k_row, long k_head, long v_row,
                            long v_head, long out_row, float scale, int f32, cudaStream_t s) {
  if (rows <= 0 || B <= 0 || Hq <= 0) return 0;
  if (D > sb::TA_MAXD || D <= 0) return -1;
  if (Hkv <= 0 || Hq % Hkv != 0 || page_size <= 0 || max_nodes <= 0 || max_nodes > sb::TREE_MAX || max_pages < 0 ||
      static_cast<long>(max_pages) * page_size > sb::TREE_MAX_KEYS)
    return (int)cudaErrorInvalidValue;
  const dim3 grid(rows, (Hq + 3) / 4), block(128);
  if (f32)
    return (int)sb::launch_pdl(sb::tree_attn_kernel<float>, grid, block, 0, s, (const float*)q, (const float*)k_cache, (const float*)v_cache,
                               table, context, cu, parents, sinks, (float*)out, B, Hq, Hkv, D, page_size, max_pages, num_slots, max_nodes,
                               q_row, q_head, k_row, k_head, v_row, v_head, out_row, scale);
  using bf = __nv_bfloat16;
  return (int)sb::launch_pdl(sb::tree_attn_kernel<bf>, grid, block, 0, s, (const bf*)q, (const bf*)k_cache, (const bf*)v_cache, table, context,
                             cu, parents, sinks, (bf*)out, B, Hq, Hkv, D, page_size, max_pages, num_slots, max_nodes, q_row, q_head, k_row,
                             k_head, v_row, v_head, out_row, scale);
}
