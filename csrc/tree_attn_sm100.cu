// Attention of drafted-token trees over the paged cache on the 5th-gen tensor cores (sm_100a). Node i of tree b stands at cache
// position context[b] + i and sees the positions in front of context[b], the nodes above it and itself (token_tree.cuh).
//
// The cache is what there is to read, once for all nodes: the nodes of a tree and the G = Hq / Hkv heads of a kv head are the rows of one
// query tile (row = node * G + head), so 128-key tiles come in once for up to 128 rows, or 256 where a tree has more.
//
//   S_g  = Q K_j^T            M 128, N 128, K D       TMEM
//   P_g  = 2^(S_g c - m)      TMEM -> registers -> bf16 in TMEM (the A operand of the next product): with heads of 64 beside the scores it came from, so
//                             that the next scores run beside this softmax; with heads of 128 there is room only over them
//   O_g += P_g V_j            M 128, N D, K 128       TMEM
//
// One CTA per SM: warps 0 and 3 issue TMA loads (a box per page and 64-wide chunk), warps 1 and 2 the products of one group each, and two
// groups of four softmax warps have one row per thread. Where a tree fits one tile the groups take key tiles in turn, as if the keys were
// split between two launches, each with its own maximum, sum and accumulator, and the epilogue joins the two; larger trees give each group
// a query tile. Either way one group's softmax runs beside the other's products.
//
// What bounds a tile is the time of a warp's softmax over its columns, not the tensor cores: so a tree of up to 64 (32) rows is put into its
// tile 2 (4) times, and each copy takes half (a quarter) of the columns, with maximum and sum of its own and zeros as weights of the others'
// columns. The copies' accumulators are joined like the groups' are.
//
// Equal shares: the key tiles of all (request, query tile pair, kv head) items are numbered through, and CTA c takes the c-th of gridDim
// equal ranges, whatever the lengths are. A range that begins or ends inside an item leaves that part's O, m, l in a workspace, and a
// second launch joins the parts in order: the same bits on every run. With `whole` each CTA takes one item, so that a row's arithmetic does
// not depend on the batch.
//
// Key and value tiles have a ring of buffers each, with a producer of its own, and the rings run on from one piece of work to the next. A wait by parity cannot tell
// one phase of a barrier from the next but one, so every waiter sees every phase or knows that the ones before it are over. Even rings give that to the groups, which
// take tiles in turn; a ring of three buffers has six barriers for it. Where pieces with one and with two query tiles follow each other, a buffer's last tile may have
// been the other group's alone: then the queries of a piece, which come once both groups' scores of the piece before are done, and the accumulators, which are
// read once its products are, stand for it.
//
// The scores of hidden nodes become -infinity by a bit mask per row, looked at in the last tiles only. Cache rows behind the last node may hold anything: pages
// behind it are fetched from outside the cache, which reads as zero, and the rest of its page is cleared in shared memory before the product of weights (zero) and
// values. So are nodes' values that are not finite: rows that see such a node become NaN, and the others stay what they are.
//
// Measured (B200, both launches, page size 16, bursts of a few ms at 1965 MHz): 64 trees of 16 nodes over 3,000 tokens, 32 / 8 heads of 128: 151 us, 0.83 of the copy
// rate; 4 trees of 64 nodes over 28,000, 32 / 4 heads of 128: 139 us, 850 TFLOP/s, tensor pipe and special functions 45 % each (172 and 161 us in calls without a
// pause, where the power cap holds the clock near 1500 MHz); 256 trees of 3 to 9 nodes over 770, 14 / 2 heads of 64: 43 us, 0.37 of the copy rate, bound by what
// lies between pieces of work (4000 cycles for a piece's 9000); one tree of 8 nodes over 1,000: 12 us.
// Every wait is bounded: on expiry the CTA records a status word, drains and returns with its TMEM freed.
#include "token_tree.cuh"

namespace sb {

constexpr int TT_THREADS = 384;
constexpr int TT_BN = 128;

template <int D, int TILES, int REP>
struct TtSmem {
  static constexpr int NCH = D / 64;                 // 128-byte chunks of the head dim
  static constexpr int Q_TILE = 128 * 128 * NCH;
  static constexpr int KV_TILE = TT_BN * 128 * NCH;  // one K or V tile
  static constexpr int K_RING = D == 64 ? 4 : 2, V_RING = D == 64 ? 6 : (TILES == 1 ? 3 : 2), RING = K_RING + V_RING;
  static constexpr int V_FULL = V_RING % 2 == 0 ? V_RING : 2 * V_RING;  // barriers of values that have come
  static constexpr int RED = REP > 1 ? 2 * 128 * 80 : 0;  // [2 groups][128 rows][16 columns + 4]: sums over the copies
  static constexpr int TABLE = (TT_THREADS * 12 + 15) / 16 * 16;
  // behind the ring: ways up [2 pieces][128 nodes], (m, l) [2 pieces][2 groups][128 rows], parents [128], requests, barriers
  static constexpr int EXTRA = 2 * 128 * 16 + 2 * 2 * 128 * 8 + 128 * 4 + RED + TABLE + 512;
  static constexpr int TOTAL = TILES * Q_TILE + RING * KV_TILE + EXTRA + 1024;  // +1024: alignment
  static constexpr int TMEM_COLS = 512;              // S_0 @0, S_1 @128, O_0 @256, O_1 @256 + D, and with heads of 64 P_0 @384, P_1 @448
  static constexpr bool APART = D == 64;             // P beside its scores, not over them: the next scores need not wait for the product
  static constexpr int P_COL = APART ? 384 : 0, P_STEP = APART ? 64 : TT_BN;
};

__device__ __forceinline__ float tt_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// mbar_wait (common.cuh) with everything behind the first few looks out of line: a step's code has to stay small, see the top of this file.
__device__ __noinline__ bool tt_wait_long(uint64_t* bar, uint32_t parity, volatile int* cta_abort, int* status, int code) {
  return mbar_wait(bar, parity, cta_abort, status, code);
}
__device__ __forceinline__ bool tt_wait(uint64_t* bar, uint32_t parity, volatile int* cta_abort, int* status, int code) {
  return mbar_try_wait(bar, parity) || tt_wait_long(bar, parity, cta_abort, status, code);
}
// A group's 128 threads make values of hidden keys harmless (0 x NaN would reach O): rows [end, to) of a tile, behind the last key, are cleared, and
// of rows [from, end), which are nodes from first_node on, 16-byte pieces that are not all finite; bad: such nodes.
template <int NCH>
__device__ __forceinline__ void tt_clean(uint8_t* v, int from, int end, int to, int first_node, int tid, uint32_t* bad) {
#pragma unroll 1
  for (int x = tid; x < (to - from) * (NCH * 8); x += 128) {
    const int vr = from + x / (NCH * 8), ch = (x / 8) % NCH;
    uint4* at = reinterpret_cast<uint4*>(v + ch * (TT_BN * 128) + vr * 128 + (x & 7) * 16);
    bool clear = vr >= end;
    if (!clear) {
      const uint4 e = *at;
      auto inf = [](uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; };
      clear = inf(e.x) || inf(e.y) || inf(e.z) || inf(e.w);
      if (clear) {
        const int node = first_node + vr - from;
        atomicOr(&bad[node >> 5], 1u << (node & 31));
        __threadfence_block();  // before the other group can read zeros: it uses the tile too where a tree has two query tiles
      }
    }
    if (clear) *at = make_uint4(0, 0, 0, 0);
  }
}
__device__ __forceinline__ void tt_barrier(int id, int nthreads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(nthreads) : "memory"); }

struct TtArgs {
  const int* table;
  const int* context;
  const int* cu;
  const int* parents;
  const float* sinks;
  __nv_bfloat16* out;
  float4* part_o;  // [2 * gridDim][4 * TILES][D / 4][32]: of 32 rows, 4 columns each: a warp has a row per lane, and a store that touches 32 lines takes it 32 cycles
  float2* part_ml;  // [2 * gridDim][128 * TILES]
  int4* plan;      // [gridDim][2]: the item that begins in this CTA and goes on in the next: its parts (0: none) and the first one's slot,
                   // kv head and number of its first node; rows of its tree: first and number
  int rows, B, Hkv, G, bq, page_shift, max_pages, num_slots, max_nodes, pairs, whole;
  long out_row;
  float c_log2;
  int* status;
};

// Sizes of a request; its nodes are rows [first, first + n) of q and out.
struct TtRequest {
  int first, ctx, n;
  __device__ __forceinline__ int keys(const TtArgs& a) const { return min(ctx + n, a.max_pages << a.page_shift); }
  __device__ __forceinline__ int tiles(const TtArgs& a) const { return n > 0 ? (keys(a) + TT_BN - 1) / TT_BN : 0; }
  // its share of what is dealt out: key tiles of all its items, or items
  template <int TILES>
  __device__ __forceinline__ int units(const TtArgs& a) const {
    const int pairs = TILES == 1 ? 1 : (n + 2 * a.bq - 1) / (2 * a.bq);
    return (a.whole ? static_cast<int>(n > 0) : tiles(a)) * a.Hkv * pairs;
  }
};
__device__ __forceinline__ TtRequest tt_request(const TtArgs& a, int b) {
  TtRequest r = {0, 0, 0};
  if (b < a.B) {
    const int first = a.cu[b], next = a.cu[b + 1], context = a.context[b];
    r.first = first;
    r.ctx = min(max(context, 0), a.max_pages << a.page_shift);
    r.n = first < 0 ? 0 : min(max(min(next, a.rows) - first, 0), a.max_nodes);
  }
  return r;
}

// One CTA's way through its range: pieces of items, each some key tiles of a (request, pair of query tiles, kv head).
template <int TILES>
struct TtWalk {
  int u, end, b, off;          // next unit of the range, its end, request and unit within it
  const TtRequest* near;       // shared memory: requests [base, base + TT_THREADS)
  int base;
  // the piece
  TtRequest r;
  int kvh, pair, tile0, nt, tiles, keys, groups;  // groups: query tiles of the pair

  __device__ __forceinline__ void look(const TtArgs& a) { r = b - base < TT_THREADS ? near[b - base] : tt_request(a, b); }
  __device__ __forceinline__ bool next(const TtArgs& a) {
    if (u >= end) return false;
    int units = r.template units<TILES>(a);
    while (off >= units) {
      off -= units;
      ++b;
      look(a);
      units = r.template units<TILES>(a);
    }
    tiles = r.tiles(a);
    keys = r.keys(a);
    const int per = a.whole ? 1 : tiles;
    const int item = off / per;
    tile0 = off - item * per;
    pair = TILES == 1 ? 0 : item / a.Hkv;
    kvh = item - pair * a.Hkv;
    const int step = min(per - tile0, end - u);
    nt = a.whole ? tiles : step;
    groups = TILES == 1 ? 1 : (r.n > (2 * pair + 1) * a.bq ? 2 : 1);
    u += step;
    off += step;
    return true;
  }
};

template <int D, int TILES, int REP>
__global__ void __launch_bounds__(TT_THREADS, 1)
tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ TtArgs a) {
  static_assert(TILES == 1 || REP == 1, "copies of a query tile where there is one");
  using S = TtSmem<D, TILES, REP>;
  constexpr int NCH = S::NCH, ROWS = 128 / REP, COLS = TT_BN / REP;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + TILES * S::Q_TILE;
  uint4* ways = reinterpret_cast<uint4*>(sKV + S::RING * S::KV_TILE);  // [2][128]
  float2* ml = reinterpret_cast<float2*>(ways + 256);                  // [2][2][128]
  float* red = reinterpret_cast<float*>(ml + 512);
  int* par = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(red) + S::RED);  // [128]
  TtRequest* near = reinterpret_cast<TtRequest*>(par + 128);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(near) + S::TABLE);
  uint64_t* q_empty = q_full + 1;
  uint64_t* full = q_empty + 1;    // [K_RING + V_FULL]
  uint64_t* empty = full + S::K_RING + S::V_FULL;  // [RING]
  uint64_t* s_full = empty + S::RING;  // [2] scores of the group are there, and every product issued before them is done
  uint64_t* p_full = s_full + 2;       // [2] the group's P is in TMEM (4 arrivals)
  uint64_t* o_full = p_full + 2;       // [2] the group's last product of the piece is done
  uint64_t* o_empty = o_full + 2;      // both accumulators have been read (8 arrivals)
  uint64_t* w_full = o_empty + 1;      // [2] ways of the piece are there
  uint64_t* w_empty = w_full + 2;      // [2] ... and have been used (8 arrivals)
  uint64_t* my_turn = w_empty + 2;     // [2] the other group's issuer is done with its step
  uint64_t* s_free = my_turn + 2;      // [2] P apart: the group has read its scores (4 arrivals)
  uint64_t* o_step = s_free + 2;       // [2] P apart: the group's product is done, P may be written again
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_step + 2);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* start = reinterpret_cast<int*>(tmem_slot + 2);  // [0] request, [1] unit within it
  int* sums = start + 2;                               // [12] units of the warps' requests
  uint32_t* bad = reinterpret_cast<uint32_t*>(sums + 12);  // [2 pieces][4] nodes with values that are not finite

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* status = a.status;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);  // one arrival per issuing warp
    for (int s = 0; s < S::K_RING + S::V_FULL; ++s) mbar_init(&full[s], 1);
    for (int s = 0; s < S::RING; ++s) mbar_init(&empty[s], 2);
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[g], 4);
      mbar_init(&o_full[g], 1);
      mbar_init(&w_full[g], 1);
      mbar_init(&w_empty[g], 8);
      mbar_init(&my_turn[g], 1);
      mbar_init(&s_free[g], 4);
      mbar_init(&o_step[g], 1);
    }
    mbar_init(o_empty, 8);
    *cta_abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::TMEM_COLS);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch_dependents();
  // ---- this CTA's range: every thread adds up some neighbouring requests, a scan gives the threads' places
  const int share = (a.B + TT_THREADS - 1) / TT_THREADS;
  const int b0 = min(static_cast<int>(threadIdx.x) * share, a.B), b1 = min(b0 + share, a.B);
  int mine = 0;
  TtRequest own = tt_request(a, b0);
  if (share == 1) {
    near[threadIdx.x] = own;
    mine = own.template units<TILES>(a);
  } else {
    for (int b = b0; b < b1; ++b) mine += tt_request(a, b).template units<TILES>(a);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sums[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < TT_THREADS / 32; ++w) {
    const int v = sums[w];
    if (w < warp) before += v;
    total += v;
  }
  before += incl - mine;
  const int nc = gridDim.x, c = blockIdx.x;
  const int per = a.whole ? 1 : total / nc, rest = a.whole ? 0 : total - per * nc;
  TtWalk<TILES> walk;
  walk.u = a.whole ? c : c * per + min(c, rest);
  walk.end = a.whole ? min(c + 1, total) : walk.u + per + (c < rest ? 1 : 0);
  if (walk.u < walk.end && before <= walk.u && walk.u < before + mine) {
    int left = walk.u - before, b = b0;
    if (share > 1)
      for (; b < b1; ++b) {
        const int units = tt_request(a, b).template units<TILES>(a);
        if (left < units) break;
        left -= units;
      }
    start[0] = b;
    start[1] = left;
  }
  __syncthreads();
  if (threadIdx.x == 0 && !a.whole) a.plan[2 * c] = make_int4(0, 0, 0, 0);  // (the same thread writes another one below where there is one)
  if (walk.u < walk.end) {
    walk.b = start[0];
    walk.off = start[1];
    walk.near = near;
    walk.base = share == 1 ? 0 : walk.b;
    if (share > 1) {
      near[threadIdx.x] = tt_request(a, walk.b + threadIdx.x);
      __syncthreads();  // (the same for all threads)
    }
    walk.look(a);
    const int page = 1 << a.page_shift, pages = TT_BN >> a.page_shift;  // of a tile

    // Steps go to the two groups in turn, and the turn runs on from piece to piece: with one query tile, key tile j of a piece belongs to group
    // (turn + j) & 1; with two, every key tile is a step of both, and group turn & 1 has the first query tile. t0: the CTA's key tiles before a piece.
    if (warp == 0 || warp == 3) {
      // -------------------------------------------------------------------- TMA producers: keys, and values with queries and ways up
      // (lane p: page p of the tile). Issuing a box costs a warp some 100 cycles, so keys and values have a warp each.
      const bool is_k = warp == 0;
      const CUtensorMap* map = is_k ? &tmK : &tmV;
      bool ok = true;
      uint32_t t0 = 0;  // tiles of the pieces before
      for (uint32_t piece = 0; ok && walk.next(a); ++piece) {
        const int nt = walk.nt;
        const int* row = a.table + static_cast<long>(walk.b) * a.max_pages;
        // a page behind the last key is fetched from behind the cache: zeros
        auto slot_of = [&](int j) {
          const int key = (walk.tile0 + j) * TT_BN + lane * page;
          return j < nt && lane < pages && key < walk.keys ? row[key >> a.page_shift] << a.page_shift : a.num_slots;
        };
        int slot0 = slot_of(0), slot1 = slot_of(1);
        if (is_k) {
          if (lane == 0 && walk.tile0 == 0 && nt < walk.tiles) {      // the item goes on in the CTAs behind this one
            const int last = walk.u - nt + walk.tiles - 1;            // unit of its last tile, and the CTA that has it
            const int owner = last < rest * (per + 1) ? last / (per + 1) : rest + (last - rest * (per + 1)) / per;
            a.plan[2 * c] = make_int4(owner - c + 1, 2 * c + (piece == 0 ? 0 : 1), walk.kvh, walk.pair * TILES * a.bq);
            a.plan[2 * c + 1] = make_int4(walk.r.first, walk.r.n, 0, 0);
          }
        } else {
          const uint32_t buf = piece & 1;
          ok = __all_sync(0xffffffffu, tt_wait(&w_empty[buf], ((piece >> 1) & 1) ^ 1, cta_abort, status, ERR_WAIT_EMPTY));
          if (!ok) break;
          const bool hides = (walk.tile0 + nt) * TT_BN > walk.r.ctx;  // the piece has keys of nodes
          if (hides) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (x * 32 + lane < walk.r.n) par[x * 32 + lane] = a.parents[walk.r.first + x * 32 + lane];
          }
          if (lane == 0) {
            ok = tt_wait(q_empty, (piece & 1) ^ 1, cta_abort, status, ERR_WAIT_EMPTY);
            if (ok) {
              mbar_arrive_expect_tx(q_full, (REP > 1 ? REP : walk.groups) * a.bq * a.G * 128 * NCH);
              const int row0 = walk.r.first + walk.pair * TILES * a.bq;
              // two query tiles, or copies of one
              for (int x = 0; x < (REP > 1 ? REP : walk.groups); ++x)
#pragma unroll
                for (int ch = 0; ch < NCH; ++ch)
                  tma_load_3d(sQ + x * (REP > 1 ? ROWS * 128 : S::Q_TILE) + ch * (128 * 128), &tmQ, q_full, ch * 64, walk.kvh * a.G,
                              row0 + (REP > 1 ? 0 : x * a.bq));
            }
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
          if (!ok) break;
          if (hides) {
            if (lane < 4) bad[buf * 4 + lane] = 0;
            __syncwarp();
            for (int i = lane; i < walk.r.n; i += 32) {
              uint32_t set[4];
              tree_way_up([&](int j) { return par[j]; }, i, set);
              ways[buf * 128 + i] = make_uint4(set[0], set[1], set[2], set[3]);
            }
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(&w_full[buf]);
        }
        for (int j = 0; j < nt; ++j) {
          const int slot2 = slot_of(j + 2);
          const uint32_t ring = is_k ? S::K_RING : S::V_RING, t = t0 + j, st = t % ring + (is_k ? 0 : S::K_RING);
          uint64_t* come = &full[is_k ? st : S::K_RING + t % S::V_FULL];
          if (lane == 0) {
            ok = tt_wait(&empty[st], (t / ring & 1) ^ 1, cta_abort, status, ERR_WAIT_EMPTY);
            if (ok) mbar_arrive_expect_tx(come, S::KV_TILE);
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
          if (!ok) break;
          if (lane < pages)
#pragma unroll
            for (int ch = 0; ch < NCH; ++ch)
              tma_load_3d(sKV + st * S::KV_TILE + ch * (TT_BN * 128) + lane * page * 128, map, come, ch * 64, walk.kvh, slot0);
          slot0 = slot1;
          slot1 = slot2;
        }
        t0 += nt;
      }
    } else if (warp < 3) {
      // -------------------------------------------------------------------- MMA issuers
      // A group's steps: scores, then (once P is there) the product, then the next step's scores, which may be the next piece's. The
      // whole warp goes through it with the same values; one lane issues. With two query tiles the issuers take turns, so that one group's
      // softmax falls beside the other's products (left to themselves they run in step and take a quarter longer, at 4 trees of 64 nodes, 32 / 4
      // heads of 128, over 28,000 keys).
      constexpr uint32_t idesc_s = make_idesc(128, TT_BN, 1, 1, 0, 0);
      constexpr uint32_t idesc_o = make_idesc(128, D, 1, 1, 0, 1);  // A = P in TMEM, B = V read MN-major
      // operands of the products come from registers that are the same for the whole warp: without the compiler knowing it each product costs some 100 cycles
      auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
      const uint32_t tmem = uniform(tmem_base);
      const uint64_t q_desc = make_smem_desc(smem_u32(sQ), 16, 1024, UMMA_SWIZZLE_128B);
      const uint64_t k_desc = make_smem_desc(smem_u32(sKV), 16, 1024, UMMA_SWIZZLE_128B);
      const uint64_t v_desc = make_smem_desc(smem_u32(sKV), TT_BN * 128, 1024, UMMA_SWIZZLE_128B);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        ok = ok && tt_wait(bar, parity, cta_abort, status, code);
        ok = __all_sync(0xffffffffu, ok);
      };
      struct Group {
        TtWalk<TILES> walk;
        uint32_t t0, turn, piece;  // tiles and turns of the pieces before, pieces
        int i;                            // the next scores: the group's i-th step of the piece
        bool more;
        // the step whose scores are issued
        uint32_t tile, of_piece;
        bool there, first, last, rows2;
      };
      auto scores = [&](Group& s, int g) {
        s.there = false;
        while (s.more) {
          const int nt = s.walk.nt;
          const bool rows2 = TILES == 2 && s.walk.groups == 2;
          const int late = (g ^ s.turn) & 1, n_my = rows2 ? nt : (nt + 1 - late) / 2, j = rows2 ? s.i : late + 2 * s.i;
          if (s.i < n_my) {
            const uint32_t t = s.t0 + j, ks = t % S::K_RING;
            if (s.i == 0) wait(q_full, s.piece & 1, ERR_WAIT_FULL);
            wait(&full[ks], t / S::K_RING & 1, ERR_WAIT_FULL);
            if (!ok) return;
            tc_fence_after();
            const uint64_t qd = q_desc + uniform(rows2 ? late : 0) * (S::Q_TILE >> 4), kd = k_desc + uniform(ks) * (S::KV_TILE >> 4);
            const uint32_t d_s = tmem + uniform(g) * TT_BN;
            const bool last = s.i + 1 == n_my;
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const int at = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
                umma_f16(d_s, qd + at, kd + at, idesc_s, k != 0 ? 1u : 0u);
              }
              umma_commit(&s_full[g]);
              umma_commit(&empty[ks]);
              if (!rows2) mbar_arrive(&empty[ks]);  // (the other group has no part in this tile)
              if (last) umma_commit(q_empty);
            }
            __syncwarp();
            s.there = true;
            s.of_piece = s.piece;
            s.tile = t;
            s.first = s.i == 0;
            s.last = last;
            s.rows2 = rows2;
            ++s.i;
            return;
          }
          if (n_my == 0) {  // no part in this piece: its queries are free as far as this group is concerned, once they are the ones in place
            wait(q_full, s.piece & 1, ERR_WAIT_FULL);
            if (!ok) return;
            if (elect_one()) mbar_arrive(q_empty);
            __syncwarp();
          }
          s.t0 += nt;
          s.turn += rows2 ? 2 * nt : nt;
          s.i = 0;
          ++s.piece;
          s.more = s.walk.next(a);
        }
      };
      constexpr bool TURNS = TILES == 2 && !S::APART;
      struct Step {
        uint32_t tile, of_piece;
        bool first, last, rows2;
      };
      auto product = [&](const Step& x, uint32_t steps, int g) {
        wait(&p_full[g], steps & 1, ERR_WAIT_TMEM_EMPTY);
        if (x.first) wait(o_empty, (x.of_piece & 1) ^ 1, ERR_WAIT_TMEM_EMPTY);  // (the accumulators of the last piece have been read)
        const uint32_t vs = x.tile % S::V_RING;
        wait(&full[S::K_RING + x.tile % S::V_FULL], x.tile / S::V_FULL & 1, ERR_WAIT_FULL);
        if (TURNS) wait(&my_turn[g], steps & 1, ERR_WAIT_EMPTY);
        if (!ok) return;
        tc_fence_after();
        const uint64_t vd = v_desc + (S::K_RING + uniform(vs)) * (S::KV_TILE >> 4);
        const uint32_t more_o = uniform(x.first ? 0u : 1u), d_o = tmem + 2 * TT_BN + uniform(g) * D, a_o = tmem + S::P_COL + uniform(g) * S::P_STEP;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < TT_BN / 16; ++k) umma_f16_ts(d_o, a_o + k * 8, vd + k * (2048 >> 4), idesc_o, k != 0 ? 1u : more_o);
          umma_commit(&empty[S::K_RING + vs]);
          if (!x.rows2) mbar_arrive(&empty[S::K_RING + vs]);
          if (S::APART) umma_commit(&o_step[g]);
          if (x.last) umma_commit(&o_full[g]);
        }
        __syncwarp();
      };
      const int g = warp - 1;
      if (TURNS && g == 1 && elect_one()) mbar_arrive(&my_turn[0]);  // group 0 begins
      __syncwarp();
      Group s = {};
      s.walk = walk;
      s.more = s.walk.next(a);
      scores(s, g);
      for (uint32_t steps = 0; ok && s.there; ++steps) {
        const Step x = {s.tile, s.of_piece, s.first, s.last, s.rows2};
        if (S::APART && !x.last) {  // the next scores run beside this step's softmax
          wait(&s_free[g], steps & 1, ERR_WAIT_TMEM_EMPTY);
          if (ok) scores(s, g);
          if (ok) product(x, steps, g);
        } else {  // (a piece's last product does not wait for the queries of the next)
          product(x, steps, g);
          if (S::APART) wait(&s_free[g], steps & 1, ERR_WAIT_TMEM_EMPTY);
          if (ok) scores(s, g);
        }
        if (TURNS && elect_one()) mbar_arrive(&my_turn[g ^ 1]);
        __syncwarp();
      }
    } else {
      // -------------------------------------------------------------------- softmax + epilogue
      const int quarter = warp & 3, g = (warp - 4) >> 2;
      const int row = quarter * 32 + lane;  // row of the query tile = TMEM lane
      const int tid = threadIdx.x & 127;
      const int copy = row / ROWS, rr = row % ROWS;  // this thread's keys of a tile: columns [copy * COLS, copy * COLS + COLS)
      const int in_tile = rr / a.G, head_in = rr - in_tile * a.G;
      const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t s_addr = lane_addr + g * TT_BN, o_addr = lane_addr + 2 * TT_BN, p_addr = lane_addr + S::P_COL + g * S::P_STEP;
      const uint64_t c2 = f2_pack(a.c_log2, a.c_log2);
      uint32_t t0 = 0, turn = 0, s_cnt = 0, o_cnt0 = 0, o_cnt1 = 0;
      bool ok = true;
      if constexpr (REP > 1 && S::APART) {  // the other copies' weights: zero for good
        const uint32_t none[16] = {};
#pragma unroll
        for (int x = 0; x < 4; ++x) tmem_st_32x16(p_addr + x * 16, none);
        tmem_st_wait();
      }
      for (uint32_t piece = 0; walk.next(a); ++piece) {  // after an expired wait the threads still meet at the barriers
        const int nt = walk.nt, ctx = walk.r.ctx;
        const bool rows2 = TILES == 2 && walk.groups == 2;
        const int late = (g ^ turn) & 1;  // the group whose turn is second
        const int qt = rows2 ? late : 0;
        const int node = (walk.pair * TILES + qt) * a.bq + in_tile;
        const bool valid = in_tile < a.bq && node < walk.r.n;
        const bool active = __any_sync(0xffffffffu, valid);  // a warp without a row only keeps step
        const bool ends = walk.tile0 + nt == walk.tiles;     // this piece has the item's last tile
        const uint32_t* way = reinterpret_cast<const uint32_t*>(&ways[(piece & 1) * 128 + (valid ? node : 0)]);
        bool have_ways = false;
        auto want_ways = [&]() {
          if (!have_ways) ok = __all_sync(0xffffffffu, ok && tt_wait(&w_full[piece & 1], (piece >> 1) & 1, cta_abort, status, ERR_WAIT_FULL));
          have_ways = true;
        };
        const int n_late = rows2 ? nt : nt / 2;  // its steps; the other one has some always
        const int n_my = rows2 ? nt : (late ? n_late : nt - n_late);
        float m_run = -INFINITY, l_run = 0.f;
        for (int i = 0; i < n_my && ok; ++i) {
          const int j = rows2 ? i : late + 2 * i;
          ok = tt_wait(&s_full[g], (s_cnt + i) & 1, cta_abort, status, ERR_WAIT_TMEM_FULL);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const int key0 = (walk.tile0 + j) * TT_BN;
          const bool masked = key0 + TT_BN > ctx;
          if (masked) {
            want_ways();
            if (!ok) break;
          }
          auto release = [&]() {  // P apart: the scores are in registers, the next ones may come
            if (S::APART) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s_free[g]);
            }
          };
          bool settled = !S::APART || s_cnt + i == 0;
          auto settle = [&]() {  // P apart: the group's last product is done, P and O may be written
            if (!settled) ok = __all_sync(0xffffffffu, ok && tt_wait(&o_step[g], (s_cnt + i - 1) & 1, cta_abort, status, ERR_WAIT_TMEM_FULL));
            settled = true;
            tc_fence_after();
          };
          if (!active) {
            release();
            settle();
          }
          if (active) {
            // hides what the row does not see of columns [32 x, 32 x + 32) of this tile: it sees keys in front of the tree, and nodes on its way up
            auto hide = [&](uint32_t (&r)[32], int x) {
              const int at = key0 + 32 * x - ctx;  // node of the first column
              uint32_t vis = 0;
              if (at <= -32) vis = 0xffffffffu;
              else if (at < 0) vis = ((1u << -at) - 1) | (way[0] << -at);
              else if (at < 128) vis = __funnelshift_r(way[at >> 5], (at >> 5) < 3 ? way[(at >> 5) + 1] : 0u, at & 31);
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if ((vis >> k & 1) == 0) r[k] = 0xff800000u;  // -infinity
            };
            auto top = [&](uint32_t (&r)[32]) {
              float m0 = __uint_as_float(r[0]), m1 = __uint_as_float(r[1]);
#pragma unroll
              for (int k = 2; k < 32; k += 2) {
                m0 = fmaxf(m0, __uint_as_float(r[k]));
                m1 = fmaxf(m1, __uint_as_float(r[k + 1]));
              }
              return fmaxf(m0, m1);
            };
            // A row of 128 columns is read twice: for its maximum the second half, then the first one, which stays in registers; the second half
            // comes back behind that (P takes the columns of the first half only).
            uint32_t ra[32], rb[32];
            float mx = -INFINITY;
            const int x0 = copy * (COLS / 32);
#pragma unroll 1
            for (int x = x0 + (COLS == 128 ? 2 : 0); x >= x0; x -= 2) {
              tmem_ld_32x32(s_addr + 32 * x, ra);
              if constexpr (COLS > 32) tmem_ld_32x32(s_addr + 32 * x + 32, rb);
              tmem_ld_wait();
              if (masked) {
                hide(ra, x);
                if constexpr (COLS > 32) hide(rb, x + 1);
              }
              mx = fmaxf(mx, COLS > 32 ? fmaxf(top(ra), top(rb)) : top(ra));
            }
            if constexpr (COLS < 128) release();
            mx *= a.c_log2;  // c > 0: the maximum commutes with the scaling
            const float m_new = fmaxf(m_run, mx);
            if (i == 0) {
              m_run = m_new;
            } else if (__any_sync(0xffffffffu, valid && m_new > m_run + 8.f)) {
              // (with P over the scores, those just read came after every earlier product, so O may be corrected)
              settle();
              const float f = m_new == -INFINITY ? 1.f : tt_exp2(m_run - m_new);
              l_run *= f;
#pragma unroll 1
              for (int c4 = 0; c4 < D / 32; ++c4) {
                uint32_t o[32];
                tmem_ld_32x32(o_addr + g * D + c4 * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                tmem_st_32x32(o_addr + g * D + c4 * 32, o);
              }
              m_run = m_new;
            }
            // ---- p = 2^(s c - m), packed to bf16; the row's sum uses the unrounded values (a row that has seen nothing yet: all 0)
            const float m_use = m_run == -INFINITY ? 0.f : m_run;
            const uint64_t nm = f2_pack(-m_use, -m_use);
            uint64_t sum[2] = {0, 0};
            auto weigh = [&](uint32_t (&r)[32], int x) {
              uint32_t pk[16];
#pragma unroll
              for (int k = 0; k < 32; k += 2) {
                float p0, p1;
                f2_unpack(f2_fma(f2_pack(__uint_as_float(r[k]), __uint_as_float(r[k + 1])), c2, nm), p0, p1);
                p0 = tt_exp2(p0);
                p1 = tt_exp2(p1);
                sum[(k >> 1) & 1] = f2_add(sum[(k >> 1) & 1], f2_pack(p0, p1));
                pk[k >> 1] = pack_bf16x2(p0, p1);
              }
              settle();
              tmem_st_32x16(p_addr + x * 16, pk);
            };
            if constexpr (REP > 1 && !S::APART) {  // the other copies' columns (over scores of this row: its own have to be in registers, as they are)
              const uint32_t none[16] = {};
#pragma unroll
              for (int x = 0; x < 4; ++x)
                if (x < x0 || x >= x0 + COLS / 32) tmem_st_32x16(p_addr + x * 16, none);
            }
#pragma unroll 1
            for (int x = x0; x < x0 + (COLS + 63) / 64 * 2; x += 2) {
              if (COLS == 128 && x > x0) {
                tmem_ld_32x32(s_addr + 32 * x, ra);
                tmem_ld_32x32(s_addr + 32 * x + 32, rb);
                tmem_ld_wait();
                release();
                if (masked) {
                  hide(ra, x);
                  hide(rb, x + 1);
                }
              }
              weigh(ra, x);
              if constexpr (COLS > 32) weigh(rb, x + 1);
            }
            float s0, s1;
            f2_unpack(f2_add(sum[0], sum[1]), s0, s1);
            l_run += s0 + s1;
          }
          if (masked) {  // values of nodes, and behind the last key: by each group that uses the tile
            const uint32_t t = t0 + j, vs = S::K_RING + t % S::V_RING;
            ok = __all_sync(0xffffffffu, tt_wait(&full[S::K_RING + t % S::V_FULL], t / S::V_FULL & 1, cta_abort, status, ERR_WAIT_FULL));
            if (!ok) break;
            const int from = max(ctx - key0, 0), end = min(walk.keys - key0, TT_BN);
            tt_clean<NCH>(sKV + vs * S::KV_TILE, from, end, (end + page - 1) & -page, key0 + from - ctx, tid, bad + (piece & 1) * 4);
            fence_proxy_async();
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g]);
        }
        s_cnt += n_my;
        bool hole = false, poisoned = false;
        if ((walk.tile0 + nt) * TT_BN > ctx) {
          want_ways();
          hole = valid && (way[0] & 1) == 0;
        }
        // ---- epilogue: with one query tile the groups (and copies) are joined, and each group writes half of the columns
        const bool all = walk.tile0 == 0 && ends;
        const int slot = 2 * c + (piece == 0 ? 0 : 1);
        const int g_first = turn & 1;  // the group whose turn was first
        const bool has0 = g_first == 0 || n_late > 0, has1 = g_first == 1 || n_late > 0;
        float f0 = 1.f, f1 = 0.f, m = m_run, l = l_run;
        if (!rows2) {
          float2* mine_ml = ml + (piece & 1) * 256;
          mine_ml[g * 128 + row] = make_float2(m_run, l_run);  // (nothing seen: -infinity, 0)
          tt_barrier(3, 256);
          m = -INFINITY;
#pragma unroll
          for (int x = 0; x < 2 * REP; ++x) m = fmaxf(m, mine_ml[(x / REP) * 128 + (x % REP) * ROWS + rr].x);
          l = 0.f;
#pragma unroll
          for (int x = 0; x < 2 * REP; ++x) {
            const float2 e = mine_ml[(x / REP) * 128 + (x % REP) * ROWS + rr];
            const float f = m == -INFINITY ? 0.f : tt_exp2(e.x - m);
            l += e.y * f;
            if (x % REP == copy) {
              if (x / REP == 0) f0 = f;
              else f1 = f;
            }
          }
        }
        if (has0 && (!rows2 || g == 0)) ok = ok && tt_wait(&o_full[0], o_cnt0 & 1, cta_abort, status, ERR_WAIT_TMEM_FULL);
        if (has1 && (!rows2 || g == 1)) ok = ok && tt_wait(&o_full[1], o_cnt1 & 1, cta_abort, status, ERR_WAIT_TMEM_FULL);
        ok = __all_sync(0xffffffffu, ok);
        o_cnt0 += has0;
        o_cnt1 += has1;
        tc_fence_after();
        if (valid && (walk.tile0 + nt) * TT_BN > ctx) {  // (every thread that looks at values of this piece's nodes has done so)
#pragma unroll
          for (int x = 0; x < 4; ++x) poisoned |= (way[x] & bad[(piece & 1) * 4 + x]) != 0;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&w_empty[piece & 1]);
        float inv = 1.f;
        if (all) {
          const int head = walk.kvh * a.G + head_in;
          if (a.sinks != nullptr && valid && l > 0.f) l += tt_exp2(a.sinks[head] * 1.4426950408889634f - m);
          inv = hole || l == 0.f ? 0.f : 1.f / l;  // (a sum that is NaN comes through)
        }
        if (poisoned) inv = __int_as_float(0x7fffffff);
        // an accumulator that nothing was added to holds anything, and a row that sees nothing is zero whatever its accumulators hold
        const float by0 = f0 * inv, by1 = f1 * inv;
        const uint32_t keep0 = has0 && by0 != 0.f ? 0xffffffffu : 0u, keep1 = has1 && by1 != 0.f ? 0xffffffffu : 0u;
        auto both = [&](uint32_t x, uint32_t y) { return fmaf(__uint_as_float(x & keep0), by0, __uint_as_float(y & keep1) * by1); };
        if constexpr (REP == 1) {
          if (ok && active) {
            // a thread writes its row: all of it, or half
            const int col0 = rows2 ? 0 : g * (D / 2), cols = rows2 ? D : D / 2;
            __nv_bfloat16* o_row = a.out + static_cast<long>(walk.r.first + node) * a.out_row + static_cast<long>(walk.kvh * a.G + head_in) * D;
            float4* p_row = a.part_o + ((static_cast<long>(slot) * TILES + qt) * 4 + quarter) * (D * 8) + lane;
            const uint32_t mine_o = o_addr + (rows2 ? g * D : 0);
#pragma unroll 1
            for (int col = col0; col < col0 + cols; col += 16) {
              uint32_t x[16], y[16];
              tmem_ld_32x16(mine_o + col, x);
              if (!rows2) tmem_ld_32x16(o_addr + D + col, y);
              tmem_ld_wait();
              float v[16];
              if (rows2) {
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = inv != 0.f ? __uint_as_float(x[k]) * inv : 0.f;
              } else {
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = both(x[k], y[k]);
              }
              if (valid && all) {
#pragma unroll
                for (int k = 0; k < 16; k += 8)
                  *reinterpret_cast<uint4*>(o_row + col + k) = make_uint4(pack_bf16x2(v[k], v[k + 1]), pack_bf16x2(v[k + 2], v[k + 3]),
                                                                          pack_bf16x2(v[k + 4], v[k + 5]), pack_bf16x2(v[k + 6], v[k + 7]));
              } else if (valid) {
#pragma unroll
                for (int k = 0; k < 16; k += 4) p_row[(col + k) * 8] = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
              }
            }
          }
        } else {
          // the copies' sums meet in shared memory, 16 columns a turn; then a thread adds up 16 / REP columns of a row, neighbours of the same
          // one where rows are written out, of the next one where parts are
          float* mine_red = red + g * (128 * 20);
          constexpr int PER = 16 / REP;
          const int o_rr = all ? tid / REP : tid % ROWS, o_col = (all ? tid % REP : tid / ROWS) * PER, o_in = o_rr / a.G, o_head = o_rr - o_in * a.G;
          const bool o_valid = ok && o_in < walk.r.n && o_in < a.bq;
          __nv_bfloat16* o_row = a.out + static_cast<long>(walk.r.first + o_in) * a.out_row + static_cast<long>(walk.kvh * a.G + o_head) * D + o_col;
          float4* p_row = a.part_o + (static_cast<long>(slot) * 4 + (o_rr >> 5)) * (D * 8) + o_col * 8 + (o_rr & 31);
          const float* from = mine_red + o_rr * 20 + o_col;
#pragma unroll 1
          for (int col = g * (D / 2); col < (g + 1) * (D / 2); col += 16) {
            if (ok && active) {
              uint32_t x[16], y[16];
              tmem_ld_32x16(o_addr + col, x);
              tmem_ld_32x16(o_addr + D + col, y);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; k += 4)
                *reinterpret_cast<float4*>(mine_red + row * 20 + k) = make_float4(both(x[k], y[k]), both(x[k + 1], y[k + 1]), both(x[k + 2], y[k + 2]),
                                                                                  both(x[k + 3], y[k + 3]));
            }
            tt_barrier(1 + g, 128);
            if (o_valid) {
              float t[PER];
#pragma unroll
              for (int k = 0; k < PER; ++k) t[k] = 0.f;
#pragma unroll
              for (int x = 0; x < REP; ++x)
#pragma unroll
                for (int k = 0; k < PER; k += 4) {
                  const float4 e = *reinterpret_cast<const float4*>(from + x * (ROWS * 20) + k);
                  t[k] += e.x; t[k + 1] += e.y; t[k + 2] += e.z; t[k + 3] += e.w;
                }
#pragma unroll
              for (int k = 0; k < PER; k += 4) {
                if (all) *reinterpret_cast<uint2*>(o_row + col + k) = make_uint2(pack_bf16x2(t[k], t[k + 1]), pack_bf16x2(t[k + 2], t[k + 3]));
                else p_row[(col + k) * 8] = make_float4(t[k], t[k + 1], t[k + 2], t[k + 3]);
              }
            }
            tt_barrier(1 + g, 128);
          }
        }
        // a node of no tree marks its row with a negative sum
        if (!all && valid && copy == 0 && (rows2 || g == 0))
          a.part_ml[static_cast<long>(slot) * (128 * TILES) + qt * 128 + rr] = make_float2(m, hole ? -1.f : l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty);
        t0 += nt;
        turn += rows2 ? 2 * nt : nt;
      }
    }
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (*cta_abort) {
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);  // let copies in flight land
    __syncthreads();
  }
  if (warp == 1) tmem_dealloc(tmem_base, S::TMEM_COLS);
}

// Joins the parts of items that were split between CTAs: out = sum_p o_p 2^(m_p - M) / sum_p l_p 2^(m_p - M), in the order of the parts. A lane has a row,
// a warp every eighth group of 4 columns. Block x looks at the item that goes on behind CTA x, if there is one.
constexpr int TT_JOIN_THREADS = 256;
template <int D, int TILES>
__global__ void __launch_bounds__(TT_JOIN_THREADS)
tree_attn_join_kernel(const __grid_constant__ TtArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int x = blockIdx.y * 32 + lane, row = x & 127, in_tile = row / a.G;
  const int4 plan = a.plan[2 * c], tree = a.plan[2 * c + 1];
  const int parts = plan.x, node = plan.w + (x >> 7) * a.bq + in_tile;
  const bool valid = parts > 0 && in_tile < a.bq && node < tree.y;
  if (!__any_sync(0xffffffffu, valid)) return;
  constexpr int NQ = D / 32;         // groups of columns
  constexpr int FLY = 16 / NQ;       // parts whose reads are under way together
  float top = -INFINITY, l = 0.f;
  float4 o[NQ];
  bool hole = false;
#pragma unroll
  for (int k = 0; k < NQ; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < parts; p0 += FLY) {
    float2 ml[FLY];
    float4 v[FLY][NQ];
#pragma unroll
    for (int i = 0; i < FLY; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      if (valid && p0 + i < parts) {
        const long slot = p0 + i == 0 ? plan.y : 2 * (c + p0 + i);  // (behind the first part: the first slot of the CTA)
        ml[i] = a.part_ml[slot * (128 * TILES) + x];
#pragma unroll
        for (int k = 0; k < NQ; ++k) v[i][k] = a.part_o[(slot * (4 * TILES) + blockIdx.y) * (D * 8) + (warp + 8 * k) * 32 + lane];
      }
    }
    float new_top = top;
#pragma unroll
    for (int i = 0; i < FLY; ++i) new_top = fmaxf(new_top, ml[i].x);
    const float zero = new_top == -INFINITY ? 0.f : new_top, keep = tt_exp2(top - zero);
    top = new_top;
    l *= keep;
#pragma unroll
    for (int k = 0; k < NQ; ++k) o[k] = make_float4(o[k].x * keep, o[k].y * keep, o[k].z * keep, o[k].w * keep);
#pragma unroll
    for (int i = 0; i < FLY; ++i) {
      if (!valid || p0 + i >= parts) break;
      const float f = tt_exp2(ml[i].x - zero);
      l += ml[i].y * f;
      hole = hole || ml[i].y < 0.f;
#pragma unroll
      for (int k = 0; k < NQ; ++k)
        o[k] = make_float4(fmaf(v[i][k].x, f, o[k].x), fmaf(v[i][k].y, f, o[k].y), fmaf(v[i][k].z, f, o[k].z), fmaf(v[i][k].w, f, o[k].w));
    }
  }
  if (!valid) return;
  const int head = plan.z * a.G + row - in_tile * a.G;
  if (a.sinks != nullptr) l += tt_exp2(a.sinks[head] * 1.4426950408889634f - top);
  const bool some = !hole && l != 0.f;  // (a sum that is NaN comes through)
  const float inv = some ? 1.f / l : 0.f;
  __nv_bfloat16* dst = a.out + static_cast<long>(tree.x + node) * a.out_row + static_cast<long>(head) * D;
#pragma unroll
  for (int k = 0; k < NQ; ++k)
    *reinterpret_cast<uint2*>(dst + (warp + 8 * k) * 4) =
        some ? make_uint2(pack_bf16x2(o[k].x * inv, o[k].y * inv), pack_bf16x2(o[k].z * inv, o[k].w * inv)) : make_uint2(0, 0);
}

template <int D, int TILES, int REP>
static int launch_tree_attn(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TtArgs& a, int ctas, cudaStream_t s) {
  using S = TtSmem<D, TILES, REP>;
  auto kern = tree_attn_tc_kernel<D, TILES, REP>;
  if (cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), S::TOTAL); e != cudaSuccess) return (int)e;
  if (cudaError_t e = launch_pdl(kern, dim3(ctas), dim3(TT_THREADS), S::TOTAL, s, tq, tk, tv, a); e != cudaSuccess) return (int)e;
  if (a.whole) return 0;
  const int rows = TILES == 1 ? a.max_nodes * a.G : 128 * TILES;
  return (int)launch_pdl(tree_attn_join_kernel<D, TILES>, dim3(ctas, (rows + 31) / 32), dim3(TT_JOIN_THREADS), 0, s, a);
}

struct TtPlan {
  int ctas, tiles, copies, bq, pairs;  // CTAs; query tiles of an item, or copies of its only one; nodes of a tile; items of a (request, kv head)
  long bytes;                          // of workspace
};
// tokens: most keys a request can have. false where the kernel does not cover the call.
static bool tree_attn_plan(int B, int Hq, int Hkv, int D, int max_nodes, long tokens, int whole, int sms, TtPlan& p) {
  if (B <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Hq / Hkv > 128 || (D != 64 && D != 128) || max_nodes <= 0 || max_nodes > TREE_MAX || tokens <= 0 || tokens > TREE_MAX_KEYS) return false;
  const int G = Hq / Hkv, rows = max_nodes * G;
  p.tiles = max_nodes > 128 / G ? 2 : 1;
  p.copies = rows <= 32 ? 4 : (rows <= 64 ? 2 : 1);
  p.bq = 128 / p.copies / G;
  p.pairs = (max_nodes + p.tiles * p.bq - 1) / (p.tiles * p.bq);
  const long items = static_cast<long>(B) * Hkv * p.pairs, units = items * ((tokens + TT_BN - 1) / TT_BN);
  if (units > 0x3fffffffl) return false;
  p.ctas = static_cast<int>(whole ? items : (units < sms ? units : sms));
  p.bytes = whole ? 16 : 32l * p.ctas + 2l * p.ctas * 128 * p.tiles * (D * 4 + 8);
  return true;
}

}  // namespace sb

// Bytes of workspace of a call, -1 where sb_tree_attn_tc does not cover it. tokens: most keys a request can have.
extern "C" int sb_tree_attn_plan(int B, int Hq, int Hkv, int D, int max_nodes, long tokens, int whole, int sms, long* bytes) {
  sb::TtPlan p;
  if (!sb::tree_attn_plan(B, Hq, Hkv, D, max_nodes, tokens, whole, sms, p)) return -1;
  *bytes = p.bytes;
  return 0;
}

// call: addresses of q, both caches, page table, context lengths, cu, parents, sinks, out, workspace, status word; then rows, B, Hq, Hkv, D, page size, pages of
// a row of the table, slots, most nodes, pitches of q (row, head), k (slot, head), v (slot, head) and out (row), whole, bytes of workspace, SMs (one
// array: a call from Python costs some 0.1 us for every argument). Everything as for sb_tree_attn (tree_attn.cu), in bf16; scale > 0; a
// 16-byte aligned workspace of the size that sb_tree_attn_plan names.
// Returns 0, a cudaError_t value, or -1 where this kernel does not cover the call: head widths other than 64 and 128, pages other than
// 16, 32, 64 and 128 tokens, more than 128 query heads on a key head, addresses or pitches that are no multiple of 16 bytes.
extern "C" int sb_tree_attn_tc(const void* call, float scale, cudaStream_t s) {
  const long long* x = static_cast<const long long*>(call);
  const int rows = x[11], B = x[12], Hq = x[13], Hkv = x[14], D = x[15], page_size = x[16], max_pages = x[17], num_slots = x[18], max_nodes = x[19];
  const long q_row = x[20], q_head = x[21], k_row = x[22], k_head = x[23], v_row = x[24], v_head = x[25], out_row = x[26];
  const int whole = x[27], sms = x[29];
  if (rows <= 0 || B <= 0) return 0;
  int shift = 4;
  while (shift < 7 && 1 << shift != page_size) ++shift;
  if (1 << shift != page_size || ((x[0] | x[1] | x[2] | x[8] | x[9]) & 15) != 0 || ((q_row | q_head | k_row | k_head | v_row | v_head | out_row) & 7) != 0 ||
      !(scale > 0.f) || num_slots <= 0 || max_pages <= 0)
    return -1;
  sb::TtPlan p;
  if (!sb::tree_attn_plan(B, Hq, Hkv, D, max_nodes, static_cast<long>(max_pages) * page_size, whole, sms, p)) return -1;
  if (p.bytes > x[28]) return (int)cudaErrorInvalidValue;
  sb::TtArgs a = {};
  a.table = reinterpret_cast<const int*>(x[3]);
  a.context = reinterpret_cast<const int*>(x[4]);
  a.cu = reinterpret_cast<const int*>(x[5]);
  a.parents = reinterpret_cast<const int*>(x[6]);
  a.sinks = reinterpret_cast<const float*>(x[7]);
  a.out = reinterpret_cast<__nv_bfloat16*>(x[8]);
  a.plan = reinterpret_cast<int4*>(x[9]);
  a.status = reinterpret_cast<int*>(x[10]);
  a.part_o = reinterpret_cast<float4*>(a.plan + 2l * p.ctas);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + 2l * p.ctas * 32 * p.tiles * D);
  a.rows = rows; a.B = B; a.Hkv = Hkv; a.G = Hq / Hkv; a.bq = p.bq; a.page_shift = shift; a.max_pages = max_pages; a.num_slots = num_slots;
  a.max_nodes = max_nodes; a.pairs = p.pairs; a.whole = whole;
  a.out_row = out_row;
  a.c_log2 = scale * 1.4426950408889634f;
  try {
    const CUtensorMap tq = sb::make_tmap_3d(reinterpret_cast<const void*>(x[0]), D, Hq, rows, q_head, q_row, 64, a.G, a.bq);
    const CUtensorMap tk = sb::make_tmap_3d(reinterpret_cast<const void*>(x[1]), D, Hkv, num_slots, k_head, k_row, 64, 1, page_size);
    const CUtensorMap tv = sb::make_tmap_3d(reinterpret_cast<const void*>(x[2]), D, Hkv, num_slots, v_head, v_row, 64, 1, page_size);
    auto by_form = [&](auto launch64, auto launch128) { return D == 64 ? launch64(tq, tk, tv, a, p.ctas, s) : launch128(tq, tk, tv, a, p.ctas, s); };
    if (p.tiles == 2) return by_form(sb::launch_tree_attn<64, 2, 1>, sb::launch_tree_attn<128, 2, 1>);
    if (p.copies == 4) return by_form(sb::launch_tree_attn<64, 1, 4>, sb::launch_tree_attn<128, 1, 4>);
    if (p.copies == 2) return by_form(sb::launch_tree_attn<64, 1, 2>, sb::launch_tree_attn<128, 1, 2>);
    return by_form(sb::launch_tree_attn<64, 1, 1>, sb::launch_tree_attn<128, 1, 1>);
  } catch (const std::exception& e) {
    sb::set_last_error(e.what());
    return (int)cudaErrorInvalidValue;
  }
}
