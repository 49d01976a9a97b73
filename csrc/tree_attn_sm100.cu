// Attention of drafted-token trees over the paged cache on the 5th-gen tensor cores (sm_100a). Node i of tree b stands at cache
// position context[b] + i and sees the positions in front of context[b], the nodes above it and itself (token_tree.cuh).
//
// The cache is what there is to read, once for all nodes: the nodes of a tree and the G = Hq / Hkv heads of a kv head are the rows of one
// query tile (row = node * G + head), so 128-key tiles come in once for up to 128 rows, or 256 where a tree has more.
//
//   S_g  = Q K_j^T            M 128, N 128, K D       TMEM
//   P_g  = 2^(S_g c - m)      TMEM -> registers -> bf16 over the scores it came from (the A operand of the next product)
//   O_g += P_g V_j            M 128, N D, K 128       TMEM
//
// One CTA per SM: warp 0 issues TMA loads (a box per page and 64-wide chunk), warp 1 the products, and two groups of four softmax warps
// have one row per thread. Where a tree fits one tile the groups take the even and the odd key tiles, as if the keys were split between
// two launches, each with its own maximum, sum and accumulator, and the epilogue joins the two; larger trees give each group
// a query tile. Either way one group's softmax runs beside the other's products.
//
// Equal shares: the key tiles of all (request, query tile pair, kv head) items are numbered through, and CTA c takes the c-th of gridDim
// equal ranges, whatever the lengths are. A range that begins or ends inside an item leaves that part's O, m, l in a workspace, and a
// second launch joins the parts in order: the same bits on every run. With `whole` each CTA takes one item, so that a row's arithmetic does
// not depend on the batch.
//
// K and V tiles share one ring in the order K0, K1, V0, K2, V1, ..., the order in which they are used, and the ring runs on from one piece
// of work to the next. The scores of hidden nodes become -infinity by a bit mask per row, looked at in the last tiles only. Cache rows behind
// the last node may hold anything: pages behind it are fetched from outside the cache, which reads as zero, and the rest of its page is
// cleared in shared memory before the product of weights (zero) and values.
// Every wait is bounded: on expiry the CTA records a status word, drains and returns with its TMEM freed.
#include "token_tree.cuh"

namespace sb {

constexpr int TT_THREADS = 320;
constexpr int TT_BN = 128;

template <int D, int TILES>
struct TtSmem {
  static constexpr int NCH = D / 64;                 // 128-byte chunks of the head dim
  static constexpr int Q_TILE = 128 * 128 * NCH;
  static constexpr int KV_TILE = TT_BN * 128 * NCH;  // one K or V tile
  static constexpr int RING = D == 64 ? 10 : (TILES == 1 ? 5 : 4);
  // behind the ring: ways up [2 groups][128 nodes], (m, l) [2 pieces][2 groups][128 rows], parents [2][128], barriers
  static constexpr int EXTRA = 2 * 128 * 16 + 2 * 2 * 128 * 8 + 2 * 128 * 4 + 512;
  static constexpr int TOTAL = TILES * Q_TILE + RING * KV_TILE + EXTRA + 1024;  // +1024: alignment
  static constexpr int TMEM_COLS = 512;              // S_0 @0, S_1 @128, O_0 @256, O_1 @256 + D
};

__device__ __forceinline__ float tt_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void tt_barrier(int id, int nthreads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(nthreads) : "memory"); }

struct TtArgs {
  const int* table;
  const int* context;
  const int* cu;
  const int* parents;
  const float* sinks;
  __nv_bfloat16* out;
  float* part_o;   // [2 * gridDim][128 * TILES][D]
  float2* part_ml;  // [2 * gridDim][128 * TILES]
  int4* plan;      // [B * Hkv * pairs]: parts of an item (0: finished), slot of the first, CTA of the first
  int rows, B, Hkv, G, bq, page_shift, max_pages, num_slots, max_nodes, pairs, whole;
  long out_row;
  float c_log2;
  int* status;
};

// Sizes of request b; its nodes are rows [first, first + n) of q and out.
struct TtRequest {
  int first, ctx, n, keys, tiles, qtiles;
};
__device__ __forceinline__ TtRequest tt_request(const TtArgs& a, int b) {
  TtRequest r;
  r.first = a.cu[b];
  const int next = a.cu[b + 1], room = a.max_pages << a.page_shift;
  r.ctx = min(max(a.context[b], 0), room);
  r.n = r.first < 0 ? 0 : min(max(min(next, a.rows) - r.first, 0), a.max_nodes);
  r.keys = min(r.ctx + r.n, room);
  r.tiles = r.n > 0 ? (r.keys + TT_BN - 1) / TT_BN : 0;
  r.qtiles = (r.n + a.bq - 1) / a.bq;
  return r;
}
template <int TILES>
__device__ __forceinline__ int tt_units(const TtArgs& a, const TtRequest& r) {
  return (a.whole ? (r.tiles > 0) : r.tiles) * a.Hkv * ((r.qtiles + TILES - 1) / TILES);
}

// One CTA's way through its range: pieces of items, each some key tiles of a (request, pair of query tiles, kv head).
template <int TILES>
struct TtWalk {
  int u, end, b, off;  // next unit of the range, its end, request and unit within it
  TtRequest r;
  // the piece
  int kvh, pair, tile0, nt, groups;  // groups: query tiles of the pair

  __device__ __forceinline__ bool next(const TtArgs& a) {
    if (u >= end) return false;
    int units = tt_units<TILES>(a, r);
    while (off >= units) {
      off -= units;
      ++b;
      r = tt_request(a, b);
      units = tt_units<TILES>(a, r);
    }
    const int per = a.whole ? 1 : r.tiles;
    const int item = off / per;
    tile0 = a.whole ? 0 : off - item * per;
    kvh = item % a.Hkv;
    pair = item / a.Hkv;
    const int step = a.whole ? 1 : min(r.tiles - tile0, end - u);
    nt = a.whole ? r.tiles : step;
    groups = TILES == 1 ? 1 : min(2, r.qtiles - 2 * pair);
    u += step;
    off += step;
    return true;
  }
};

template <int D, int TILES>
__global__ void __launch_bounds__(TT_THREADS, 1)
tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ TtArgs a) {
  using S = TtSmem<D, TILES>;
  constexpr int NCH = S::NCH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + TILES * S::Q_TILE;
  uint4* ways = reinterpret_cast<uint4*>(sKV + S::RING * S::KV_TILE);  // [2][128]
  float2* ml = reinterpret_cast<float2*>(ways + 256);                  // [2][2][128]
  int* par = reinterpret_cast<int*>(ml + 512);                         // [2][128]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(par + 256);
  uint64_t* q_empty = q_full + 1;
  uint64_t* full = q_empty + 1;    // [RING]
  uint64_t* empty = full + S::RING;
  uint64_t* s_full = empty + S::RING;  // [2] scores of the group are there, and every product issued before them is done
  uint64_t* p_full = s_full + 2;       // [2] the group's P is in TMEM (4 arrivals)
  uint64_t* o_full = p_full + 2;       // [2] the group's last product of the piece is done
  uint64_t* o_empty = o_full + 2;      // both accumulators have been read (8 arrivals)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_empty + 1);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* start = reinterpret_cast<int*>(tmem_slot + 2);  // [0] request, [1] unit within it
  int* sums = start + 2;                               // [10] units of the warps' requests

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* status = a.status;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < S::RING; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[g], 4);
      mbar_init(&o_full[g], 1);
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
  for (int b = b0; b < b1; ++b) mine += tt_units<TILES>(a, tt_request(a, b));
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
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  before += incl - mine;
  const int nc = gridDim.x, c = blockIdx.x;
  const int per = a.whole ? 1 : total / nc, rest = a.whole ? 0 : total - per * nc;
  TtWalk<TILES> walk;
  walk.u = a.whole ? c : c * per + min(c, rest);
  walk.end = a.whole ? min(c + 1, total) : walk.u + per + (c < rest ? 1 : 0);
  if (walk.u < walk.end && before <= walk.u && walk.u < before + mine) {
    int left = walk.u - before, b = b0;
    for (; b < b1; ++b) {
      const int units = tt_units<TILES>(a, tt_request(a, b));
      if (left < units) break;
      left -= units;
    }
    start[0] = b;
    start[1] = left;
  }
  __syncthreads();
  if (walk.u < walk.end) {
    walk.b = start[0];
    walk.off = start[1];
    walk.r = tt_request(a, walk.b);
    const int page = 1 << a.page_shift, pages = TT_BN >> a.page_shift;  // of a tile

    if (warp == 0) {
      // -------------------------------------------------------------------- TMA producer (lane p: page p of the tile)
      bool ok = true;
      uint32_t half = 0;  // halves issued so far
      auto fetch = [&](const CUtensorMap* map, int slot0) {
        const uint32_t st = half % S::RING;
        if (lane == 0) {
          ok = mbar_wait(&empty[st], ((half / S::RING) & 1) ^ 1, cta_abort, status, ERR_WAIT_EMPTY);
          if (ok) mbar_arrive_expect_tx(&full[st], S::KV_TILE);
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (ok && lane < pages)
#pragma unroll
          for (int ch = 0; ch < NCH; ++ch)
            tma_load_3d(sKV + st * S::KV_TILE + ch * (TT_BN * 128) + lane * page * 128, map, &full[st], ch * 64, walk.kvh, slot0);
        ++half;
      };
      for (uint32_t piece = 0; ok && walk.next(a); ++piece) {
        const int* row = a.table + static_cast<long>(walk.b) * a.max_pages;
        // a page behind the last key is fetched from behind the cache: zeros
        auto slot_of = [&](int j) {
          const int key = (walk.tile0 + j) * TT_BN + lane * page;
          return j < walk.nt && lane < pages && key < walk.r.keys ? row[key >> a.page_shift] << a.page_shift : a.num_slots;
        };
        int s0 = slot_of(0), s1 = slot_of(1);
        if (lane == 0) {
          ok = mbar_wait(q_empty, (piece & 1) ^ 1, cta_abort, status, ERR_WAIT_EMPTY);
          if (ok) {
            mbar_arrive_expect_tx(q_full, walk.groups * a.bq * a.G * 128 * NCH);
            const int node0 = walk.r.first + walk.pair * TILES * a.bq;
            for (int g = 0; g < walk.groups; ++g)
#pragma unroll
              for (int ch = 0; ch < NCH; ++ch)
                tma_load_3d(sQ + g * S::Q_TILE + ch * (128 * 128), &tmQ, q_full, ch * 64, walk.kvh * a.G, node0 + g * a.bq);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!ok) break;
        fetch(&tmK, s0);
        for (int j = 0; j < walk.nt && ok; ++j) {
          const int s2 = slot_of(j + 2);
          if (j + 1 < walk.nt) fetch(&tmK, s1);
          if (ok) fetch(&tmV, s0);
          s0 = s1;
          s1 = s2;
        }
      }
    } else if (warp == 1) {
      // -------------------------------------------------------------------- MMA issuer
      if (lane == 0) {
        constexpr uint32_t idesc_s = make_idesc(128, TT_BN, 1, 1, 0, 0);
        constexpr uint32_t idesc_o = make_idesc(128, D, 1, 1, 0, 1);  // A = P in TMEM, B = V read MN-major
        bool ok = true;
        uint32_t half0 = 0, p_cnt[2] = {0, 0};
        for (uint32_t piece = 0; ok && walk.next(a); ++piece) {
          const int nt = walk.nt;
          const bool rows2 = walk.groups == 2;
          auto k_half = [&](int j) { return half0 + (j == 0 ? 0 : 2 * j - 1); };
          auto v_half = [&](int j) { return half0 + (j + 1 < nt ? 2 * j + 2 : 2 * nt - 1); };
          auto wait_half = [&](uint32_t h) {
            ok = ok && mbar_wait(&full[h % S::RING], (h / S::RING) & 1, cta_abort, status, ERR_WAIT_FULL);
            if (ok) tc_fence_after();
          };
          auto issue_s = [&](int g, int j) {
            const uint32_t q_addr = smem_u32(sQ + (rows2 ? g * S::Q_TILE : 0)), k_addr = smem_u32(sKV + (k_half(j) % S::RING) * S::KV_TILE);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t at = (k >> 2) * (128 * 128) + (k & 3) * 32;
              umma_f16(tmem_base + g * TT_BN, make_smem_desc(q_addr + at, 16, 1024, UMMA_SWIZZLE_128B),
                       make_smem_desc(k_addr + at, 16, 1024, UMMA_SWIZZLE_128B), idesc_s, k != 0 ? 1u : 0u);
            }
            umma_commit(&s_full[g]);
          };
          auto issue_o = [&](int g, int j, bool first) {
            const uint32_t v_addr = smem_u32(sKV + (v_half(j) % S::RING) * S::KV_TILE);
#pragma unroll
            for (int k = 0; k < TT_BN / 16; ++k)
              umma_f16_ts(tmem_base + 2 * TT_BN + g * D, tmem_base + g * TT_BN + k * 8,
                          make_smem_desc(v_addr + k * 2048, TT_BN * 128, 1024, UMMA_SWIZZLE_128B), idesc_o, (!first || k != 0) ? 1u : 0u);
          };
          auto wait_p = [&](int g) {
            ok = ok && mbar_wait(&p_full[g], p_cnt[g]++ & 1, cta_abort, status, ERR_WAIT_TMEM_EMPTY);
            if (ok) tc_fence_after();
          };
          auto free_half = [&](uint32_t h) { umma_commit(&empty[h % S::RING]); };
          ok = mbar_wait(q_full, piece & 1, cta_abort, status, ERR_WAIT_FULL);
          wait_half(k_half(0));
          if (!ok) break;
          issue_s(0, 0);
          if (rows2) {
            issue_s(1, 0);
            free_half(k_half(0));
            if (nt == 1) umma_commit(q_empty);
          } else {
            free_half(k_half(0));
            if (nt > 1) {
              wait_half(k_half(1));
              if (!ok) break;
              issue_s(1, 1);
              free_half(k_half(1));
            }
            if (nt <= 2) umma_commit(q_empty);
          }
          for (int j = 0; j < nt && ok; ++j) {
            wait_half(v_half(j));
            if (rows2) {
              for (int g = 0; g < 2 && ok; ++g) {
                wait_p(g);
                if (j == 0 && g == 0) ok = ok && mbar_wait(o_empty, (piece & 1) ^ 1, cta_abort, status, ERR_WAIT_TMEM_EMPTY);
                if (!ok) break;
                tc_fence_after();
                issue_o(g, j, j == 0);
                if (j + 1 == nt) umma_commit(&o_full[g]);
                if (j + 1 < nt) {
                  wait_half(k_half(j + 1));
                  if (!ok) break;
                  issue_s(g, j + 1);
                }
              }
              if (!ok) break;
              free_half(v_half(j));
              if (j + 1 < nt) free_half(k_half(j + 1));
              if (j + 2 == nt) umma_commit(q_empty);
            } else {
              const int g = j & 1;
              wait_p(g);
              if (j == 0) ok = ok && mbar_wait(o_empty, (piece & 1) ^ 1, cta_abort, status, ERR_WAIT_TMEM_EMPTY);
              if (!ok) break;
              tc_fence_after();
              issue_o(g, j, j < 2);
              free_half(v_half(j));
              if (j + 2 >= nt) umma_commit(&o_full[g]);
              if (j + 2 < nt) {
                wait_half(k_half(j + 2));
                if (!ok) break;
                issue_s(g, j + 2);
                free_half(k_half(j + 2));
                if (j + 3 == nt) umma_commit(q_empty);
              }
            }
          }
          half0 += 2 * nt;
        }
      }
    } else {
      // -------------------------------------------------------------------- softmax + epilogue
      const int quarter = warp & 3, g = (warp - 2) >> 2;
      const int row = quarter * 32 + lane;  // row of the query tile = TMEM lane
      const int tid = (threadIdx.x - 64) & 127;
      const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t s_addr = lane_addr + g * TT_BN;
      const uint64_t c2 = f2_pack(a.c_log2, a.c_log2);
      uint32_t half0 = 0, s_cnt = 0, o_cnt[2] = {0, 0};
      bool ok = true;
      for (uint32_t piece = 0; walk.next(a); ++piece) {  // after an expired wait the threads still meet at the barriers
        const int nt = walk.nt, keys = walk.r.keys, ctx = walk.r.ctx;
        const bool rows2 = walk.groups == 2;
        const int in_tile = row / a.G, node = (walk.pair * TILES + (rows2 ? g : 0)) * a.bq + in_tile;
        const int head = walk.kvh * a.G + row - in_tile * a.G;
        const bool valid = in_tile < a.bq && node < walk.r.n;
        const bool ends = walk.tile0 + nt == walk.r.tiles;                  // this piece has the item's last tile
        const bool hides = (walk.tile0 + nt) * TT_BN > ctx;                  // ... or another one with nodes
        bool hole = false;
        if (hides) {
          tt_barrier(1 + g, 128);  // the last piece's ways have been read
          if (tid < walk.r.n) par[g * 128 + tid] = a.parents[walk.r.first + tid];
          tt_barrier(1 + g, 128);
          uint32_t set[4] = {0, 0, 0, 0};
          if (tid < walk.r.n) tree_way_up([&](int i) { return par[g * 128 + i]; }, tid, set);
          ways[g * 128 + tid] = make_uint4(set[0], set[1], set[2], set[3]);
          tt_barrier(1 + g, 128);
          hole = valid && (ways[g * 128 + node].x & 1) == 0;
        }
        const int step = rows2 ? 1 : 2;
        const int n_my = rows2 ? nt : (nt + 1 - g) / 2;
        float m_run = -INFINITY, l_run = 0.f;
        for (int i = 0; i < n_my && ok; ++i) {
          const int j = rows2 ? i : g + i * step;
          ok = mbar_wait(&s_full[g], (s_cnt + i) & 1, cta_abort, status, ERR_WAIT_TMEM_FULL);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const int key0 = (walk.tile0 + j) * TT_BN;
          const bool masked = key0 + TT_BN > ctx;
          uint32_t vis[4];
          if (masked) {
            // bit i: key key0 + i: in front of the tree, or a node on the way up
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&ways[g * 128 + (valid ? node : 0)]);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int at = key0 + 32 * x - ctx;  // node of the word's first bit
              uint32_t v = 0;
              if (at <= -32) v = 0xffffffffu;
              else if (at < 0) v = ((1u << -at) - 1) | (w[0] << -at);
              else if (at < 128) v = __funnelshift_r(w[at >> 5], (at >> 5) < 3 ? w[(at >> 5) + 1] : 0u, at & 31);
              vis[x] = v;
            }
          }
          uint32_t r[4][32];
          auto load = [&](int c4) { tmem_ld_32x32(s_addr + c4 * 32, r[c4]); };
          auto hide = [&](int c4) {
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if ((vis[c4] >> x & 1) == 0) r[c4][x] = 0xff800000u;  // -infinity
          };
          float mx4[4];
          auto row_max = [&](int c4) {
            if (masked) hide(c4);
            mx4[c4] = __uint_as_float(r[c4][0]);
#pragma unroll
            for (int x = 1; x < 32; ++x) mx4[c4] = fmaxf(mx4[c4], __uint_as_float(r[c4][x]));
          };
          load(3);
          load(0);
          tmem_ld_wait();
          load(1);
          load(2);
          row_max(3);
          row_max(0);
          tmem_ld_wait();
          row_max(1);
          row_max(2);
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.c_log2;  // c > 0: the maximum commutes with the scaling
          const float m_new = fmaxf(m_run, mx);
          if (i == 0) {
            m_run = m_new;
          } else if (__any_sync(0xffffffffu, valid && m_new > m_run + 8.f)) {
            // (the scores just read came after every earlier product, so O may be corrected)
            const float f = m_new == -INFINITY ? 1.f : tt_exp2(m_run - m_new);
            l_run *= f;
            const uint32_t o_addr = lane_addr + 2 * TT_BN + g * D;
#pragma unroll 1
            for (int c4 = 0; c4 < D / 32; ++c4) {
              uint32_t o[32];
              tmem_ld_32x32(o_addr + c4 * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st_32x32(o_addr + c4 * 32, o);
            }
            m_run = m_new;
          }
          // ---- p = 2^(s c - m), packed to bf16; the row's sum uses the unrounded values (a row that has seen nothing yet: all 0)
          const float m_use = m_run == -INFINITY ? 0.f : m_run;
          const uint64_t nm = f2_pack(-m_use, -m_use);
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4) {
            if (c4 == 1) load(3);  // (P takes the columns of the first two quarters only)
            if (c4 == 3) {
              tmem_ld_wait();
              if (masked) hide(3);
            }
            uint32_t pk[16];
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              float p0, p1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c4][x]), __uint_as_float(r[c4][x + 1])), c2, nm), p0, p1);
              p0 = tt_exp2(p0);
              p1 = tt_exp2(p1);
              sum[(x >> 1) & 1] = f2_add(sum[(x >> 1) & 1], f2_pack(p0, p1));
              pk[x >> 1] = pack_bf16x2(p0, p1);
            }
            tmem_st_32x16(s_addr + c4 * 16, pk);
          }
          if (ends && j + 1 == nt && (!rows2 || g == 0) && (keys & (TT_BN - 1)) != 0) {
            // value rows behind the last key: the rest of its page is cleared (0 x NaN would reach O)
            const uint32_t h = half0 + 2 * nt - 1;
            ok = __all_sync(0xffffffffu, mbar_wait(&full[h % S::RING], (h / S::RING) & 1, cta_abort, status, ERR_WAIT_FULL));
            if (!ok) break;
            const int from = keys & (TT_BN - 1), to = min(TT_BN, (from + page - 1) & -page);
            uint8_t* v = sKV + (h % S::RING) * S::KV_TILE;
            for (int x = tid; x < (to - from) * NCH * 8; x += 128) {
              const int rr = from + x / (NCH * 8), ch = (x / 8) % NCH;
              *reinterpret_cast<uint4*>(v + ch * (TT_BN * 128) + rr * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g]);
          float s0, s1;
          f2_unpack(f2_add(sum[0], sum[1]), s0, s1);
          l_run += s0 + s1;
        }
        s_cnt += n_my;
        // ---- epilogue
        const int n_of1 = rows2 ? nt : nt / 2;  // key tiles of group 1 (group 0 always has some)
        const bool all = walk.tile0 == 0 && ends;
        const int slot = 2 * static_cast<int>(blockIdx.x) + (piece == 0 ? 0 : 1);
        float f0 = 1.f, f1 = 0.f, m = m_run, l = l_run;
        int col0 = 0, col1 = D;
        if (!rows2) {
          float2* mine_ml = ml + (piece & 1) * 256;
          mine_ml[g * 128 + row] = make_float2(m_run, l_run);
          tt_barrier(3, 256);
          const float2 x0 = mine_ml[row], x1 = mine_ml[128 + row];  // (a group that saw nothing: -infinity, 0)
          m = fmaxf(x0.x, x1.x);
          f0 = m == -INFINITY ? 0.f : tt_exp2(x0.x - m);
          f1 = m == -INFINITY ? 0.f : tt_exp2(x1.x - m);
          l = x0.y * f0 + x1.y * f1;
          col0 = g * (D / 2);
          col1 = col0 + D / 2;
        }
        if (ok && (!rows2 || g == 0)) ok = mbar_wait(&o_full[0], o_cnt[0] & 1, cta_abort, status, ERR_WAIT_TMEM_FULL);
        if (ok && n_of1 > 0 && (!rows2 || g == 1)) ok = mbar_wait(&o_full[1], o_cnt[1] & 1, cta_abort, status, ERR_WAIT_TMEM_FULL);
        ok = __all_sync(0xffffffffu, ok);
        o_cnt[0] += 1;
        o_cnt[1] += n_of1 > 0 ? 1 : 0;
        if (ok) {
          tc_fence_after();
          float inv = 1.f;
          if (all) {
            if (a.sinks != nullptr && valid && l > 0.f) l += tt_exp2(a.sinks[head] * 1.4426950408889634f - m);
            inv = (l > 0.f && !hole) ? 1.f / l : 0.f;
          }
          __nv_bfloat16* o_row = a.out + static_cast<long>(walk.r.first + node) * a.out_row + static_cast<long>(head) * D;
          float* p_row = a.part_o + (static_cast<long>(slot) * (128 * TILES) + (rows2 ? g * 128 : 0) + row) * D;
#pragma unroll 1
          for (int c = col0; c < col1; c += 32) {
            uint32_t x[32], y[32];
            tmem_ld_32x32(lane_addr + 2 * TT_BN + (rows2 ? g * D : 0) + c, x);
            if (!rows2 && n_of1 > 0) tmem_ld_32x32(lane_addr + 2 * TT_BN + D + c, y);
            tmem_ld_wait();
            if (!rows2) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                x[i] = __float_as_uint(__uint_as_float(x[i]) * f0 + (n_of1 > 0 ? __uint_as_float(y[i]) * f1 : 0.f));
            }
            if (!valid) continue;
            if (all) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (inv > 0.f) {
                  v.x = pack_bf16x2(__uint_as_float(x[8 * i]) * inv, __uint_as_float(x[8 * i + 1]) * inv);
                  v.y = pack_bf16x2(__uint_as_float(x[8 * i + 2]) * inv, __uint_as_float(x[8 * i + 3]) * inv);
                  v.z = pack_bf16x2(__uint_as_float(x[8 * i + 4]) * inv, __uint_as_float(x[8 * i + 5]) * inv);
                  v.w = pack_bf16x2(__uint_as_float(x[8 * i + 6]) * inv, __uint_as_float(x[8 * i + 7]) * inv);
                }
                *reinterpret_cast<uint4*>(o_row + c + 8 * i) = v;
              }
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<uint4*>(p_row + c + 4 * i) = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            }
          }
          // a node of no tree marks its row with an infinite maximum
          if (!all && valid && (rows2 || g == 0))
            a.part_ml[static_cast<long>(slot) * (128 * TILES) + (rows2 ? g * 128 : 0) + row] = make_float2(hole ? INFINITY : m, l);
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty);
        if (walk.tile0 == 0 && g == 0 && tid == 0) {
          int4 p = make_int4(0, slot, blockIdx.x, 0);
          if (!all) {
            const int last = walk.u - nt + walk.r.tiles - 1;  // unit of the item's last tile, and the CTA that has it
            const int owner = last < rest * (per + 1) ? last / (per + 1) : rest + (last - rest * (per + 1)) / per;
            p.x = owner - static_cast<int>(blockIdx.x) + 1;
          }
          a.plan[(static_cast<long>(walk.b) * a.Hkv + walk.kvh) * a.pairs + walk.pair] = p;
        }
        half0 += 2 * nt;
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

// Joins the parts of items that were split between CTAs: out = sum_p o_p 2^(m_p - M) / sum_p l_p 2^(m_p - M), a warp per row, in the order of the parts.
template <int D, int TILES>
__global__ void __launch_bounds__(128)
tree_attn_join_kernel(const __grid_constant__ TtArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int item = blockIdx.x, pair = item % a.pairs, kvh = item / a.pairs % a.Hkv, b = item / (a.pairs * a.Hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TtRequest req = tt_request(a, b);
  const int first = req.first, n = req.n;
  if (pair * TILES * a.bq >= n) return;
  const int4 plan = a.plan[item];
  if (plan.x == 0) return;
  constexpr int V = D / 32;  // channels of a lane
  for (int x = blockIdx.y * 16 + warp; x < min(blockIdx.y * 16 + 16, 128 * TILES); x += 4) {
    const int row = x & 127, in_tile = row / a.G, node = (pair * TILES + (x >> 7)) * a.bq + in_tile;
    if (in_tile >= a.bq || node >= n) continue;
    // part p: in slot plan.y, or the first slot of the CTA behind
    auto at = [&](int p) { return static_cast<long>(p == 0 ? plan.y : 2 * (plan.z + p)) * (128 * TILES) + x; };
    float top = -INFINITY;
    for (int p = lane; p < plan.x; p += 32) top = fmaxf(top, a.part_ml[at(p)].x);
    top = warp_max(top);
    float l = 0.f, o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.f;
    if (top != INFINITY) {
      for (int p0 = 0; p0 < plan.x; p0 += 32) {
        const float2 mine = p0 + lane < plan.x ? a.part_ml[at(p0 + lane)] : make_float2(-INFINITY, 0.f);
        const float f = mine.x == -INFINITY ? 0.f : tt_exp2(mine.x - top);
        l += warp_sum(mine.y * f);
        const int count = min(32, plan.x - p0);
#pragma unroll 4
        for (int p = 0; p < count; ++p) {
          const float fp = __shfl_sync(0xffffffffu, f, p);
          const float* src = a.part_o + at(p0 + p) * D + lane * V;
          if constexpr (V == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src);
            o[0] = fmaf(v.x, fp, o[0]); o[1] = fmaf(v.y, fp, o[1]); o[2] = fmaf(v.z, fp, o[2]); o[3] = fmaf(v.w, fp, o[3]);
          } else {
            const float2 v = *reinterpret_cast<const float2*>(src);
            o[0] = fmaf(v.x, fp, o[0]); o[1] = fmaf(v.y, fp, o[1]);
          }
        }
      }
    }
    const int head = kvh * a.G + row - in_tile * a.G;
    if (a.sinks != nullptr && l > 0.f) l += tt_exp2(a.sinks[head] * 1.4426950408889634f - top);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    __nv_bfloat16* dst = a.out + static_cast<long>(first + node) * a.out_row + static_cast<long>(head) * D + lane * V;
    if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
    else *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(o[0] * inv, o[1] * inv);
  }
}

template <int D, int TILES>
static int launch_tree_attn(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TtArgs& a, int ctas, cudaStream_t s) {
  using S = TtSmem<D, TILES>;
  auto kern = tree_attn_tc_kernel<D, TILES>;
  if (cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), S::TOTAL); e != cudaSuccess) return (int)e;
  if (cudaError_t e = launch_pdl(kern, dim3(ctas), dim3(TT_THREADS), S::TOTAL, s, tq, tk, tv, a); e != cudaSuccess) return (int)e;
  if (a.whole) return 0;
  const int rows = (a.max_nodes + a.bq - 1) / a.bq == 1 ? a.max_nodes * a.G : 128 * TILES;
  return (int)launch_pdl(tree_attn_join_kernel<D, TILES>, dim3(a.B * a.Hkv * a.pairs, (rows + 15) / 16), dim3(128), 0, s, a);
}

}  // namespace sb

// Work of a call: CTAs, query tiles of an item and bytes of workspace, as sb_tree_attn_tc wants them. tokens: most keys a request can have.
extern "C" int sb_tree_attn_plan(int B, int Hq, int Hkv, int D, int max_nodes, long tokens, int whole, int sms, int* ctas, int* tiles, long* bytes) {
  if (B <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Hq / Hkv > 128 || (D != 64 && D != 128) || max_nodes <= 0 || max_nodes > sb::TREE_MAX) return -1;
  const int G = Hq / Hkv, bq = 128 / G, qtiles = (max_nodes + bq - 1) / bq;
  *tiles = qtiles > 1 ? 2 : 1;
  const long items = static_cast<long>(B) * Hkv * ((qtiles + *tiles - 1) / *tiles);
  const long units = items * ((tokens + sb::TT_BN - 1) / sb::TT_BN);
  if (units > 0x3fffffffl) return -1;
  *ctas = static_cast<int>(whole ? items : (units < sms ? units : sms));
  const long parts = whole ? 0 : 2l * *ctas * 128 * *tiles;
  *bytes = items * 16 + parts * (D * 4 + 8);
  return 0;
}

// Arguments as for sb_tree_attn (tree_attn.cu), bf16. scale > 0. work: 16-byte aligned workspace of the size that sb_tree_attn_plan names.
// Returns 0, a cudaError_t value, or -1 where this kernel does not cover the call: head widths other than 64 and 128, pages other than
// 16, 32, 64 and 128 tokens, more than 128 query heads on a key head, addresses or pitches that are no multiple of 16 bytes.
extern "C" int sb_tree_attn_tc(const void* q, const void* k_cache, const void* v_cache, const int* table, const int* context, const int* cu,
                               const int* parents, const float* sinks, void* out, int rows, int B, int Hq, int Hkv, int D, int page_size,
                               int max_pages, int num_slots, int max_nodes, long q_row, long q_head, long k_row, long k_head, long v_row,
                               long v_head, long out_row, float scale, int whole, void* work, long work_bytes, int sms, int* status,
                               cudaStream_t s) {
  if (rows <= 0 || B <= 0) return 0;
  int shift = 4;
  while (shift < 7 && 1 << shift != page_size) ++shift;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
                          reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(work);
  if (1 << shift != page_size || (bases & 15) != 0 || ((q_row | q_head | k_row | k_head | v_row | v_head | out_row) & 7) != 0 || !(scale > 0.f) ||
      num_slots <= 0 || max_pages <= 0)
    return -1;
  int ctas = 0, tiles = 0;
  long bytes = 0;
  if (sb_tree_attn_plan(B, Hq, Hkv, D, max_nodes, static_cast<long>(max_pages) * page_size, whole, sms, &ctas, &tiles, &bytes) != 0) return -1;
  if (bytes > work_bytes) return (int)cudaErrorInvalidValue;
  const int G = Hq / Hkv, bq = 128 / G, qtiles = (max_nodes + bq - 1) / bq;
  const long items = static_cast<long>(B) * Hkv * ((qtiles + tiles - 1) / tiles);
  const long parts = whole ? 0 : 2l * ctas * 128 * tiles;
  sb::TtArgs a = {};
  a.table = table; a.context = context; a.cu = cu; a.parents = parents; a.sinks = sinks;
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.plan = reinterpret_cast<int4*>(work);
  a.part_o = reinterpret_cast<float*>(a.plan + items);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + parts * D);
  a.rows = rows; a.B = B; a.Hkv = Hkv; a.G = G; a.bq = bq; a.page_shift = shift; a.max_pages = max_pages; a.num_slots = num_slots; a.max_nodes = max_nodes;
  a.pairs = (qtiles + tiles - 1) / tiles;
  a.whole = whole;
  a.out_row = out_row;
  a.c_log2 = scale * 1.4426950408889634f;
  a.status = status;
  try {
    const CUtensorMap tq = sb::make_tmap_3d(q, D, Hq, rows, q_head, q_row, 64, G, bq);
    const CUtensorMap tk = sb::make_tmap_3d(k_cache, D, Hkv, num_slots, k_head, k_row, 64, 1, page_size);
    const CUtensorMap tv = sb::make_tmap_3d(v_cache, D, Hkv, num_slots, v_head, v_row, 64, 1, page_size);
    if (D == 64) return tiles == 1 ? sb::launch_tree_attn<64, 1>(tq, tk, tv, a, ctas, s) : sb::launch_tree_attn<64, 2>(tq, tk, tv, a, ctas, s);
    return tiles == 1 ? sb::launch_tree_attn<128, 1>(tq, tk, tv, a, ctas, s) : sb::launch_tree_attn<128, 2>(tq, tk, tv, a, ctas, s);
  } catch (const std::exception& e) {
    sb::set_last_error(e.what());
    return (int)cudaErrorInvalidValue;
  }
}
