// Acceptance of drafted-token trees (sm_100a): which drafted tokens the model itself sampled, and their keys and values in place.
//
// From the root, the walk goes to the lowest-numbered child whose drafted token is the one that the row of the node it stands on
// sampled, as long as there is one. The tokens sampled on that path are the request's next tokens. Node i of a tree was written to
// cache position context + i; path[j] >= j, and the rows of the accepted nodes move to context + j, in every layer's keys and values.
//
// One launch: grid (request, part of the cache). Every CTA does its request's walk for itself: one warp holds the nodes, four to a
// lane, and finds the next one by ballot, about 40 cycles a step. Then a thread owns 16-byte columns of (slab, row) and moves all of the
// path's rows there, up to eight reads ahead of the writes. That is safe within a thread: sources increase along the path, so
// a row that is written is never the source of a later step, and the source of an earlier step has been read. What
// bounds it is latency: reading the tree, the walk, one read and one write of a row. Measured (B200): 64 trees of 16 nodes, 36 layers of 8 heads of
// 128: 12.8 us for 29 MB; 256 trees of up to 64 nodes, 24 layers of 2 heads of 64: 7.2 us; one tree of 8: 3.4 us.
#include "token_tree.cuh"

namespace sb {

constexpr int AC_THREADS = 256;
constexpr int AC_SLABS = 128;

struct AcceptSlabs {
  uint8_t* base[AC_SLABS];  // each the first of `layers` slabs, `step` bytes apart
  long step;
  int layers, count, slots, row_units, unit;  // slabs in all; a row: row_units pieces of `unit` bytes (1, 2, 4, 8 or 16)
  long row_bytes;           // pitch of a slot
};

template <typename U>
__device__ __forceinline__ void accept_move(const AcceptSlabs& c, const int* src, const int* dst, int moves, int part, int parts) {
  const long total = static_cast<long>(c.count) * c.row_units;
  for (long x = static_cast<long>(part) * AC_THREADS + threadIdx.x; x < total; x += static_cast<long>(parts) * AC_THREADS) {
    const int slab = static_cast<int>(x / c.row_units), col = static_cast<int>(x - static_cast<long>(slab) * c.row_units);
    uint8_t* base = c.base[slab / c.layers] + slab % c.layers * c.step + static_cast<long>(col) * sizeof(U);
    for (int j0 = 0; j0 < moves; j0 += 8) {
      U held[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < moves) held[j] = *reinterpret_cast<const U*>(base + src[j0 + j] * c.row_bytes);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < moves) *reinterpret_cast<U*>(base + dst[j0 + j] * c.row_bytes) = held[j];
    }
  }
}

__global__ void __launch_bounds__(AC_THREADS)
tree_accept_kernel(const int* __restrict__ sampled, const int* __restrict__ drafted, const int* __restrict__ parents,
                   const int* __restrict__ cu, int* __restrict__ path, int* __restrict__ tokens, int* __restrict__ count, int rows, int max_nodes,
                   const __grid_constant__ AcceptSlabs slabs, const int* __restrict__ table, const int* __restrict__ context,
                   int page_size, int max_pages, int writes) {
  __shared__ int way[TREE_MAX], said[TREE_MAX];
  __shared__ int src[TREE_MAX], dst[TREE_MAX];
  __shared__ int steps, moves;
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x, lane = threadIdx.x & 31;
  const int first = cu[b], n = first < 0 ? 0 : min(max(min(cu[b + 1], rows) - first, 0), max_nodes);
  if (threadIdx.x < 32) {
    int up[4], draft[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int i = w * 32 + lane;
      up[w] = i > 0 && i < n ? parents[first + i] : -1;
      if (up[w] >= i) up[w] = -1;
      draft[w] = i < n ? drafted[first + i] : 0;
      if (i < n) said[i] = sampled[first + i];
    }
    __syncwarp();
    int here = n > 0 ? 0 : -1, j = 0;
    while (here >= 0) {
      const int tok = said[here];
      if (lane == 0) way[j] = here;
      ++j;
      int next = -1;
#pragma unroll
      for (int w = 3; w >= 0; --w) {
        const unsigned hit = __ballot_sync(0xffffffffu, up[w] == here && draft[w] == tok);
        if (hit != 0) next = w * 32 + __ffs(hit) - 1;
      }
      here = next;
    }
    if (lane == 0) steps = j;
  }
  __syncthreads();
  const int taken = steps;
  if (writes && blockIdx.y == 0) {
    for (int j = threadIdx.x; j < max_nodes; j += AC_THREADS) {
      path[static_cast<long>(b) * max_nodes + j] = j < taken ? way[j] : -1;
      tokens[static_cast<long>(b) * max_nodes + j] = j < taken ? said[way[j]] : -1;
    }
    if (threadIdx.x == 0) count[b] = taken;
  }
  if (slabs.count == 0) return;
  // ---- rows to move, in path order
  if (threadIdx.x < 32) {
    int m = 0;
    for (int j0 = 0; j0 < taken; j0 += 32) {
      const int j = j0 + lane;
      bool go = j < taken && way[j] != j;
      int from = 0, to = 0;
      if (go) {
        const long ps = static_cast<long>(context[b]) + way[j], pd = static_cast<long>(context[b]) + j;
        go = context[b] >= 0 && ps < static_cast<long>(max_pages) * page_size;
        if (go) {
          const int* row = table + static_cast<long>(b) * max_pages;
          const long s = static_cast<long>(row[ps / page_size]) * page_size + ps % page_size;
          const long d = static_cast<long>(row[pd / page_size]) * page_size + pd % page_size;
          go = s >= 0 && s < slabs.slots && d >= 0 && d < slabs.slots;
          from = static_cast<int>(s);
          to = static_cast<int>(d);
        }
      }
      const unsigned all = __ballot_sync(0xffffffffu, go);
      if (go) {
        const int at = m + __popc(all & ((1u << lane) - 1));
        src[at] = from;
        dst[at] = to;
      }
      m += __popc(all);
    }
    if (lane == 0) moves = m;
  }
  __syncthreads();
  if (slabs.unit == 16) accept_move<uint4>(slabs, src, dst, moves, blockIdx.y, gridDim.y);
  else if (slabs.unit == 8) accept_move<uint2>(slabs, src, dst, moves, blockIdx.y, gridDim.y);
  else if (slabs.unit == 4) accept_move<uint32_t>(slabs, src, dst, moves, blockIdx.y, gridDim.y);
  else if (slabs.unit == 2) accept_move<uint16_t>(slabs, src, dst, moves, blockIdx.y, gridDim.y);
  else accept_move<uint8_t>(slabs, src, dst, moves, blockIdx.y, gridDim.y);
}

}  // namespace sb

// call: addresses of sampled, drafted, parents, cu, path, tokens, count, page table and context lengths; then rows, B, most nodes, page size, pages of a row
// of the table, whether to write path, tokens and count, SMs, slabs behind each address, bytes between them, slots, pieces of a row, bytes of a
// piece (1, 2, 4, 8 or 16; addresses and pitches are multiples of it), bytes from one slot to the next, number of addresses, and the addresses, each the first of
// so many slabs. path, tokens: [B, max_nodes], -1 behind the accepted nodes; count: [B]. No address: nothing is moved.
extern "C" int sb_tree_accept(const void* call, cudaStream_t s) {
  const long long* x = static_cast<const long long*>(call);
  auto ints = [&](int i) { return reinterpret_cast<int*>(x[i]); };
  const int rows = x[9], B = x[10], max_nodes = x[11], page_size = x[12], max_pages = x[13], writes = x[14], sms = x[15], layers = x[16], n = x[22];
  if (B <= 0) return 0;
  if (max_nodes <= 0 || max_nodes > sb::TREE_MAX || n < 0 || n > sb::AC_SLABS || (n > 0 && (page_size <= 0 || layers <= 0))) return (int)cudaErrorInvalidValue;
  sb::AcceptSlabs c = {};
  for (int i = 0; i < n; ++i) c.base[i] = reinterpret_cast<uint8_t*>(x[23 + i]);
  c.layers = layers;
  c.step = x[17];
  c.count = n * layers;
  c.slots = static_cast<int>(x[18]);
  c.row_units = static_cast<int>(x[19]);
  c.unit = static_cast<int>(x[20]);
  c.row_bytes = x[21];
  if (n > 0) {
    bool fits = c.unit > 0 && c.unit <= 16 && (c.unit & (c.unit - 1)) == 0 && c.row_bytes % c.unit == 0 && c.step % c.unit == 0;
    for (int i = 0; i < n; ++i) fits = fits && x[23 + i] % c.unit == 0;
    if (!fits) return (int)cudaErrorInvalidValue;
  }
  const long all = (static_cast<long>(c.count) * c.row_units + sb::AC_THREADS - 1) / sb::AC_THREADS;
  const long want = (4L * sms + B - 1) / B;
  const int parts = static_cast<int>(all < 1 ? 1 : (all < want ? all : want));
  return (int)sb::launch_pdl(sb::tree_accept_kernel, dim3(B, parts), dim3(sb::AC_THREADS), 0, s, ints(0), ints(1), ints(2), ints(3), ints(4), ints(5), ints(6),
                             rows, max_nodes, c, ints(7), ints(8), page_size, max_pages, writes);
}
