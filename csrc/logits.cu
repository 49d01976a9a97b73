// Logits before sampling: penalties for tokens of the text, biases, and the mask of a grammar, in one pass (sm_100a).
//
//   x = logits[r, t];  c = times that t was answered with (or drafted on the way to node r), seen = c > 0 or t is in the prompt
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - c * frequency - (c > 0) * presence + sum of the biases of t;   x = -inf where the mask's bit of t is 0
//
// Nearly all logits of a row are only copied or masked. So a call of some size takes two launches: `logits_count_kernel` counts each request's text in a
// hash table in shared memory and lists the few tokens that were used or have a bias, `logits_row_kernel` copies and masks the rows at the rate of
// memory and puts in the listed ones while their lines are near. A request needs no table of the vocabulary's size that would have to be
// kept, cleared and read, only its text. (Putting them in behind the whole copy cost 55 us of 195 at 763 rows of 151936: single
// words to lines that had left the L2.) A small call takes one launch, `logits_kernel`, that keeps a chunk of a row in registers while it counts.
// Biases of a token are added up in list order: nothing depends on an order of arrival. Logits that the mask hides are not read.
// Everything is worked out in fp32 and rounded once. What bounds it: reading and writing the logits, 16 bytes a thread and access; a row that
// does not start on such a boundary is cut at the boundaries all the same, and its two ends go element by element.
// Measured (B200): 256 rows of 151936 fp32, texts of 1150: 64 us, of which the rows take 46 (6.8 TB/s) and counting, a chain of atomics and loads in few CTAs, the
// rest; 763 rows of 61 trees with masks: 171 us, 0.81 of the copy rate; one row: 3.7 us. As the engine's decode steps call it, in place and with texts in a tensor of
// 32769 columns: 45 us for those 256 rows (in place only the listed tokens are written, all are read).
#include "token_tree.cuh"

namespace sb {

constexpr int LG_THREADS = 256;
constexpr int LG_BUCKETS = 1024;

struct LogitsArgs {
  const void* in;
  void* out;
  const int* tokens;      // [S, text] tokens of each request: prompt, then answer
  const int* lengths;     // [S]
  const int* prompts;     // [S] leading tokens that are prompt, or null: none
  const float* repetition;  // [S] each, or null
  const float* frequency;
  const float* presence;
  const int* bias_ids;    // [S, biases], negative: unused
  const float* bias_values;
  const int* allowed;     // [R, words]
  const int* drafted;     // [R] trees of drafted tokens, or null: row r is request r
  const int* parents;
  const int* cu;          // [S + 1]
  long in_row, out_row, tokens_row, bias_row, allowed_row;
  int rows, requests, vocab, text, biases;
  int chunks;             // of the vocabulary
  int penal;
  // what logits_count_kernel leaves for logits_row_kernel: of each row of a tree the nodes on its way and its request; of each request the tokens
  // to work out, what there is of them and their biases, by bucket of 2^bucket_shift tokens
  int listed, bucket_shift, lists;  // lists of a request: token t is in list t % lists
  long list_room;
  uint4* row_way;
  int* row_request;
  int* list_start;        // [S, lists, buckets + 1]
  int2* list;             // [S, lists, list_room] token, what there is of it
  float* list_bias;       // where it has a bias
};

// 16-byte pieces of a row. A row's places are numbered from the 16-byte boundary at or in front of its start, so that place p is token p - off.
template <typename T, int NV>
struct Pieces {
  static constexpr int E = 16 / sizeof(T);  // tokens of a piece
  static_assert(NV * E <= 32, "a thread's mask bits are one word");
  const T* in;
  T* out;
  bool same;      // out is cut at the same tokens
  int base;       // token of the thread's CTA's first place
  uint32_t bits;  // of the mask, E for each piece
  uint4 x[NV];

  __device__ __forceinline__ int token(int i) const { return base + (i * LG_THREADS + threadIdx.x) * E; }
  __device__ __forceinline__ void load(const LogitsArgs& a, int r, int first_place) {
    in = reinterpret_cast<const T*>(a.in) + r * a.in_row;
    out = reinterpret_cast<T*>(a.out) + r * a.out_row;
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
    same = static_cast<int>((reinterpret_cast<uintptr_t>(out) & 15) / sizeof(T)) == off;
    base = first_place - off;
    bits = 0xffffffffu;
    if (a.allowed != nullptr) {
      const int* allowed = a.allowed + r * a.allowed_row;
      const int words = (a.vocab + 31) / 32;
      bits = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int t0 = token(i);
        if (t0 + E <= 0 || t0 >= a.vocab) continue;
        const int lo = t0 >> 5, hi = min((t0 + E - 1) >> 5, words - 1);  // (t0 below 0: an arithmetic shift, word -1)
        const uint32_t w0 = lo < 0 ? 0u : static_cast<uint32_t>(allowed[lo]), w1 = hi == lo ? w0 : static_cast<uint32_t>(allowed[hi]);
        bits |= (__funnelshift_r(w0, w1, t0 & 31) & ((1u << E) - 1)) << (i * E);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int t0 = token(i);
      x[i] = make_uint4(0, 0, 0, 0);
      if (shown(i) == 0) continue;
      if (t0 >= 0 && t0 + E <= a.vocab) {
        x[i] = *reinterpret_cast<const uint4*>(in + t0);
      } else {
        T* e = reinterpret_cast<T*>(&x[i]);
#pragma unroll
        for (int k = 0; k < E; ++k)
          if (t0 + k >= 0 && t0 + k < a.vocab) e[k] = in[t0 + k];
      }
    }
  }
  __device__ __forceinline__ uint32_t shown(int i) const { return bits >> (i * E) & ((1u << E) - 1); }
  __device__ __forceinline__ void store(const LogitsArgs& a, int i) {
    const int t0 = token(i);
    if (same && t0 >= 0 && t0 + E <= a.vocab) {
      *reinterpret_cast<uint4*>(out + t0) = x[i];
    } else {
      const T* e = reinterpret_cast<const T*>(&x[i]);
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (t0 + k >= 0 && t0 + k < a.vocab) out[t0 + k] = e[k];
    }
  }
};

// What a token's logit becomes.
__device__ __forceinline__ float lg_used(float v, bool seen, int times, float rep, float freq, float pres, float bias) {
  if (seen) v = v > 0.f ? v / rep : v * rep;
  if (times > 0) v = v - freq * static_cast<float>(times) - pres;
  return v + bias;
}

// What there is of a token: in the prompt, has a bias, was drafted, its bias is listed more than once, one of the bias's entries has been seen to; and how many
// times it was answered with. lg_text: each token of a request's text.
enum : int { LG_PROMPT = 1 << 30, LG_BIAS = 1 << 29, LG_DRAFT = 1 << 28, LG_TWICE = 1 << 27, LG_TAKEN = 1 << 26, LG_TIMES = LG_TAKEN - 1 };
constexpr int LG_FLY = 4;  // tokens whose reads are under way together
template <typename F>
__device__ __forceinline__ void lg_text(const LogitsArgs& a, int req, int threads, const F& each) {
  const int* text = a.tokens + req * a.tokens_row;
  const int len = max(min(a.lengths[req], a.text), 0);
  for (int i0 = threadIdx.x; i0 < len; i0 += LG_FLY * threads) {
    int t[LG_FLY];  // tokens at i0 + x threads; -1: none (or one outside the vocabulary)
#pragma unroll
    for (int x = 0; x < LG_FLY; ++x) {
      t[x] = i0 + x * threads < len ? text[i0 + x * threads] : -1;
      if (static_cast<unsigned>(t[x]) >= static_cast<unsigned>(a.vocab)) t[x] = -1;
    }
    each(i0, t);
  }
}

// Biases of a request, once all entries are marked (lg_mark): `each` gets every token with a place, once, and its bias. The first entry of a token to come stands for it;
// where there are more of them a warp goes through the list for that token and adds up in the list's order.
__device__ __forceinline__ void lg_mark(int* at) {
  if (atomicOr(at, LG_BIAS) & LG_BIAS) atomicOr(at, LG_TWICE);
}
template <typename Place, typename F>
__device__ __forceinline__ void lg_biases(const int* ids, const float* values, int K, int threads, const Place& place, const F& each) {
  const int lane = threadIdx.x & 31;
  for (int i0 = threadIdx.x - lane; i0 < K; i0 += threads) {
    const int i = i0 + lane, id = i < K ? ids[i] : -1;
    int* at = place(id);
    const int what = at != nullptr ? atomicOr(at, LG_TAKEN) : LG_TAKEN;
    const bool first = (what & LG_TAKEN) == 0;
    float bias = first ? values[i] : 0.f;
    for (uint32_t more = __ballot_sync(0xffffffffu, first && (what & LG_TWICE)); more != 0; more &= more - 1) {
      const int src = __ffs(more) - 1, t = __shfl_sync(0xffffffffu, id, src);
      float sum = 0.f;
      for (int j0 = 0; j0 < K; j0 += 32) {
        const int j = j0 + lane;
        const bool same = j < K && ids[j] == t;
        const float v = same ? values[j] : 0.f;
        for (uint32_t hit = __ballot_sync(0xffffffffu, same); hit != 0; hit &= hit - 1) sum += __shfl_sync(0xffffffffu, v, __ffs(hit) - 1);
      }
      if (lane == src) bias = sum;
    }
    if (first) each(id, at, what, bias);
  }
}

__device__ __forceinline__ void lg_prefetch(const void* at) { asm volatile("prefetch.global.L1 [%0];" ::"l"(at)); }

// ---------------------------------------------------------------- one launch: CHUNK tokens of a row, CHUNK / 256 a thread
template <typename T, int CHUNK>
__global__ void __launch_bounds__(LG_THREADS)
logits_kernel(const __grid_constant__ LogitsArgs a) {
  using Row = Pieces<T, CHUNK / LG_THREADS * static_cast<int>(sizeof(T)) / 16>;
  constexpr int E = Row::E, NV = CHUNK / LG_THREADS / E;
  __shared__ __align__(16) int count[CHUNK];
  __shared__ __align__(16) float bias[CHUNK];
  __shared__ int tree_p[TREE_MAX], tree_t[TREE_MAX];
  __shared__ int found;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int r = blockIdx.x / a.chunks, chunk = blockIdx.x - r * a.chunks;
  Row x;
  x.load(a, r, chunk * CHUNK);
  // ---- whose row it is
  int req = r, first = 0, n = 0;
  if (a.cu != nullptr) {
    if (tid == 0) found = -1;
    __syncthreads();
    for (int b = tid; b < a.requests; b += LG_THREADS)
      if (max(a.cu[b], 0) <= r && r < a.cu[b + 1]) found = b;
    __syncthreads();
    req = found;
    if (req < 0) return;  // behind the last tree: left as it is
    first = a.cu[req];
    n = first < 0 ? 0 : min(min(a.cu[req + 1], a.rows) - first, TREE_MAX);
  }
  const float rep = a.repetition != nullptr ? a.repetition[req] : 1.f;
  const float freq = a.frequency != nullptr ? a.frequency[req] : 0.f;
  const float pres = a.presence != nullptr ? a.presence[req] : 0.f;
  const bool counts = a.penal && (rep != 1.f || freq != 0.f || pres != 0.f);
  // ---- tables of this chunk
  const int base = x.base;
  auto place = [&](int t) { return t >= 0 && t < a.vocab && t >= base && t - base < CHUNK ? t - base : -1; };
  for (int i = tid; i < CHUNK / 4; i += LG_THREADS) {
    reinterpret_cast<int4*>(count)[i] = make_int4(0, 0, 0, 0);
    reinterpret_cast<int4*>(bias)[i] = make_int4(0, 0, 0, 0);
  }
  if (counts)
    for (int i = tid; i < n; i += LG_THREADS) {
      tree_p[i] = a.parents[first + i];
      tree_t[i] = a.drafted[first + i];
    }
  __syncthreads();
  if (counts) {
    const int prompt = a.prompts != nullptr ? a.prompts[req] : 0;
    lg_text(a, req, LG_THREADS, [&](int i0, const int (&t)[LG_FLY]) {
#pragma unroll
      for (int x = 0; x < LG_FLY; ++x)
        if (const int at = place(t[x]); at >= 0) {
          if (i0 + x * LG_THREADS < prompt) atomicOr(&count[at], LG_PROMPT);
          else atomicAdd(&count[at], 1);
        }
    });
    if (r - first < n) {  // the drafted tokens on the way to this row
      uint32_t set[4];
      tree_way_up([&](int j) { return tree_p[j]; }, r - first, set);
      if (tid > 0 && tid < n) {
        uint32_t word = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (tid >> 5 == w) word = set[w];
        const int at = place(tree_t[tid]);
        if ((word >> (tid & 31) & 1) && at >= 0) atomicAdd(&count[at], 1);
      }
    }
  }
  int any_bias = 0;
  const int K = a.biases;
  const int* ids = a.bias_ids + req * a.bias_row;
  const float* values = a.bias_values + req * a.bias_row;
  for (int i = tid; i < K; i += LG_THREADS)
    if (const int at = place(ids[i]); at >= 0) {
      lg_mark(&count[at]);
      any_bias = 1;
    }
  any_bias = __syncthreads_or(any_bias);
  if (any_bias) {
    lg_biases(ids, values, K, LG_THREADS, [&](int t) { const int at = place(t); return at >= 0 ? &count[at] : nullptr; },
              [&](int, int* at, int, float sum) { bias[at - count] = sum; });
    __syncthreads();
  }
  // ---- the row
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * LG_THREADS + tid) * E, t0 = x.token(i);
    if (t0 + E <= 0 || t0 >= a.vocab) continue;
    T* e = reinterpret_cast<T*>(&x.x[i]);
    const uint32_t shown = x.shown(i);
#pragma unroll
    for (int q = 0; q < E; q += 4) {
      const int4 c4 = *reinterpret_cast<const int4*>(count + at + q);
      const int cs[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = cs[k];
        float v = static_cast<float>(e[q + k]);
        if (c != 0) v = lg_used(v, (c & (LG_PROMPT | LG_TIMES)) != 0, c & LG_TIMES, rep, freq, pres, any_bias ? bias[at + q + k] : 0.f);
        if ((shown >> (q + k) & 1) == 0) v = -INFINITY;
        e[q + k] = static_cast<T>(v);
      }
    }
    x.store(a, i);
  }
}

// ---------------------------------------------------------------- two launches: count; then copy, mask and put in what was counted
// Lists the tokens of a request that were used, drafted or have a bias, by bucket of the vocabulary. They are counted in a hash table of HASH places
// in shared memory (linear probing, at most three quarters full); a longer text is counted in a table of 2 HASH tokens of the vocabulary at a time.
template <int HASH, int THREADS>
__global__ void __launch_bounds__(THREADS, HASH == 8192 ? 2 : 1)
logits_count_kernel(const __grid_constant__ LogitsArgs a) {
  extern __shared__ __align__(16) int tables[];
  int* keys = tables;          // [HASH] token, -1: empty
  int* hashed = tables + HASH;  // [HASH] what there is of it
  __shared__ int tree_p[TREE_MAX], tree_t[TREE_MAX];
  __shared__ int start[LG_BUCKETS + 1];  // places in the list: how many of a bucket, then where the next one goes
  __shared__ int sums[32];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, req = blockIdx.x / a.lists, part = blockIdx.x - req * a.lists;
  int first = 0, until = 0, n = 0;
  if (a.cu != nullptr) {
    first = a.cu[req];
    until = min(a.cu[req + 1], a.rows);
    n = first < 0 ? 0 : max(min(until - first, TREE_MAX), 0);
  }
  const float rep = a.repetition != nullptr ? a.repetition[req] : 1.f;
  const float freq = a.frequency != nullptr ? a.frequency[req] : 0.f;
  const float pres = a.presence != nullptr ? a.presence[req] : 0.f;
  // (read whether they count or not: one wait for memory instead of two)
  const int all_len = a.penal ? max(min(a.lengths[req], a.text), 0) : 0, all_prompt = a.penal && a.prompts != nullptr ? a.prompts[req] : 0;
  const int K = a.biases;
  const int* ids = a.bias_ids + req * a.bias_row;
  const float* values = a.bias_values + req * a.bias_row;
  if (tid < K) {
    lg_prefetch(ids + tid);
    lg_prefetch(values + tid);
  }
  const bool counts = a.penal && (rep != 1.f || freq != 0.f || pres != 0.f);
  const int len = counts ? all_len : 0, prompt = counts ? all_prompt : 0;
#pragma unroll
  for (int x = 0; x < LG_FLY; ++x)
    if (tid + x * THREADS < len) lg_prefetch(a.tokens + req * a.tokens_row + tid + x * THREADS);
  const bool direct = static_cast<long>(len) + K + n > HASH / 4 * 3;
  for (int i = tid; i < n; i += THREADS) {
    tree_p[i] = a.parents[first + i];
    tree_t[i] = a.drafted[first + i];
  }
  __syncthreads();
  if (a.cu != nullptr && part == 0)
    for (int r = max(first, 0) + tid; r < until; r += THREADS) {  // rows of the tree: whose they are, and the nodes on the way to them (the root is the text's last token)
      uint32_t set[4] = {0, 0, 0, 0};
      if (r - first < n) tree_way_up([&](int j) { return tree_p[j]; }, r - first, set);
      a.row_way[r] = make_uint4(set[0] & ~1u, set[1], set[2], set[3]);
      a.row_request[r] = req;
    }
  const int buckets = ((a.vocab - 1) >> a.bucket_shift) + 1;
  int* list_start = a.list_start + static_cast<long>(blockIdx.x) * (buckets + 1);
  int2* list = a.list + static_cast<long>(blockIdx.x) * a.list_room;
  float* list_bias = a.list_bias + static_cast<long>(blockIdx.x) * a.list_room;
  auto ours = [&](int t) { return static_cast<unsigned>(t) < static_cast<unsigned>(a.vocab) && (t & (a.lists - 1)) == part; };
  const int passes = direct ? (a.vocab + 2 * HASH - 1) / (2 * HASH) : 1;
  for (int i = tid; i < buckets; i += THREADS) start[i] = 0;
  int listed = 0;  // by the passes before
  for (int pass = 0; pass < passes; ++pass) {
    const int base = pass * 2 * HASH;
    const int4 empty = direct ? make_int4(0, 0, 0, 0) : make_int4(-1, -1, -1, -1);
    for (int i = tid; i < HASH / 4; i += THREADS) {
      reinterpret_cast<int4*>(keys)[i] = empty;
      reinterpret_cast<int4*>(hashed)[i] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
    // ---- what there is of each token. came: it was not there before; in the hash table the thread that brought it lists it
    auto hash = [&](int t) { return static_cast<int>((static_cast<unsigned>(t) * 2654435761u) >> 16) & (HASH - 1); };  // Knuth's multiplicative hashing
    auto look = [&](int at) { return *static_cast<volatile int*>(&keys[at]); };
    auto probe = [&](int t, int at, bool& came) -> int {  // the place of t, from place `at` on
      came = false;
      while (true) {
        int was = look(at);
        if (was == -1) {
          was = atomicCAS(&keys[at], -1, t);
          came = was == -1;
          if (came) atomicAdd(&start[t >> a.bucket_shift], 1);
        }
        if (was == -1 || was == t) return at;
        at = (at + 1) & (HASH - 1);
      }
    };
    auto place = [&](int t, bool& came) -> int* {
      came = false;
      if (!ours(t)) return nullptr;
      if (direct) return t >= base && t - base < 2 * HASH ? tables + (t - base) : nullptr;
      return &hashed[probe(t, hash(t), came)];
    };
    uint32_t brought = 0, brought_x = 0;  // of this thread's tokens of the text, one bit each (at most 12); of drafted nodes and biases
    bool came;
    if (counts) {
      int batch = 0;
      lg_text(a, req, THREADS, [&](int i0, const int (&t)[LG_FLY]) {
        // a step for all tokens at a time: nearly all of them are found, or find an empty place, at the first look
        int at[LG_FLY], was[LG_FLY];
        if (!direct) {
#pragma unroll
          for (int x = 0; x < LG_FLY; ++x) {
            at[x] = hash(t[x]);
            was[x] = ours(t[x]) ? look(at[x]) : -1;
          }
#pragma unroll
          for (int x = 0; x < LG_FLY; ++x)
            if (ours(t[x]) && was[x] == -1) {
              was[x] = atomicCAS(&keys[at[x]], -1, t[x]);
              if (was[x] == -1) {
                was[x] = t[x];
                brought |= 1u << (batch * LG_FLY + x);
                atomicAdd(&start[t[x] >> a.bucket_shift], 1);
              }
            }
#pragma unroll
          for (int x = 0; x < LG_FLY; ++x)
            if (ours(t[x]) && was[x] != t[x]) {
              at[x] = probe(t[x], at[x], came);
              if (came) brought |= 1u << (batch * LG_FLY + x);
            }
        }
#pragma unroll
        for (int x = 0; x < LG_FLY; ++x) {
          if (!ours(t[x]) || (direct && (t[x] < base || t[x] - base >= 2 * HASH))) continue;
          int* what = direct ? tables + (t[x] - base) : hashed + at[x];
          if (i0 + x * THREADS < prompt) atomicOr(what, LG_PROMPT);
          else atomicAdd(what, 1);
        }
        batch = min(batch + 1, 3);  // (more than two batches: the direct table, which needs no marks)
      });
      if (tid > 0 && tid < n)
        if (int* at = place(tree_t[tid], came); at != nullptr) {
          atomicOr(at, LG_DRAFT);
          if (came) brought_x = 1;
        }
    }
    for (int i = tid; i < K; i += THREADS)
      if (int* at = place(ids[i], came); at != nullptr) lg_mark(at);
    __syncthreads();
    // ---- by bucket: how many there are, where each bucket begins, then the tokens (in any order within a bucket)
    if (direct) {
      for (int at = tid; at < 2 * HASH; at += THREADS)
        if (tables[at] != 0) atomicAdd(&start[(base + at) >> a.bucket_shift], 1);
      __syncthreads();
    }
    const int b0 = direct ? base >> a.bucket_shift : 0, b1 = direct ? min(buckets, (base + 2 * HASH) >> a.bucket_shift) : buckets;  // of this pass
    for (int from = b0; from < b1; from += THREADS) {
      const int b = from + tid, mine_b = b < b1 ? start[b] : 0;
      int incl = mine_b;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) sums[warp] = incl;
      __syncthreads();
      int before = listed, total = 0;
      for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += sums[w];
        total += sums[w];
      }
      if (b < b1) start[b] = list_start[b] = before + incl - mine_b;
      listed += total;
      __syncthreads();
    }
    if (pass + 1 == passes && tid == 0) list_start[buckets] = listed;
    auto put = [&](int t, int what, float bias) {
      const int at = atomicAdd(&start[t >> a.bucket_shift], 1);
      list[at] = make_int2(t, what);
      if (what & LG_BIAS) list_bias[at] = bias;
    };
    if (direct) {
      for (int at = tid; at < 2 * HASH; at += THREADS)
        if (const int what = tables[at]; what != 0 && (what & LG_BIAS) == 0) put(base + at, what, 0.f);
    } else if (counts) {
      int batch = 0;
      lg_text(a, req, THREADS, [&](int, const int (&t)[LG_FLY]) {
        const uint32_t own = brought >> (batch++ * LG_FLY);
        int at[LG_FLY], to[LG_FLY], what[LG_FLY];
#pragma unroll
        for (int x = 0; x < LG_FLY; ++x) at[x] = own >> x & 1 ? hash(t[x]) : -1;
#pragma unroll
        for (int x = 0; x < LG_FLY; ++x)
          while (at[x] >= 0 && look(at[x]) != t[x]) at[x] = (at[x] + 1) & (HASH - 1);
#pragma unroll
        for (int x = 0; x < LG_FLY; ++x) {
          what[x] = at[x] >= 0 ? hashed[at[x]] : LG_BIAS;
          to[x] = (what[x] & LG_BIAS) == 0 ? atomicAdd(&start[t[x] >> a.bucket_shift], 1) : -1;
        }
#pragma unroll
        for (int x = 0; x < LG_FLY; ++x)
          if (to[x] >= 0) list[to[x]] = make_int2(t[x], what[x]);
      });
      if (brought_x)
        if (const int what = *place(tree_t[tid], came); (what & LG_BIAS) == 0) put(tree_t[tid], what, 0.f);
    }
    lg_biases(ids, values, K, THREADS, [&](int t) { return place(t, came); }, [&](int t, int*, int what, float bias) { put(t, what, bias); });
    if (pass + 1 < passes) __syncthreads();
  }
  pdl_launch_dependents();  // not before: rows that wait for the lists would slow the counting down (a tenth of the call at 256 rows of 151936)
}

// Copies and masks a chunk of a row, then puts in the logits of the listed tokens (their lines have just been here).
template <typename T>
__global__ void __launch_bounds__(LG_THREADS)
logits_row_kernel(const __grid_constant__ LogitsArgs a) {
  constexpr int NV = 4, E = 16 / sizeof(T), CHUNK = NV * E * LG_THREADS;
  // The rows were there before the launch in front of this one, which has waited for them: only the lists have to be waited for.
  if (!a.listed) pdl_wait();
  const int tid = threadIdx.x;
  const int r = blockIdx.x / a.chunks, chunk = blockIdx.x - r * a.chunks;
  if (a.cu != nullptr && (r < a.cu[0] || r >= a.cu[a.requests])) {  // not a row of a tree: left as it is
    pdl_wait();
    return;
  }
  Pieces<T, NV> x;
  x.load(a, r, chunk * CHUNK);
  if (a.listed) pdl_wait();
  pdl_launch_dependents();
  const int lo = max(x.base, 0), hi = min(x.base + CHUNK, a.vocab);  // the chunk's tokens
  // the request's lists share the threads
  int req = r, from = 0, until = 0;
  const int share = LG_THREADS / max(a.lists, 1), mine = tid / share;
  long at = 0;
  if (a.listed && lo < hi) {
    if (a.cu != nullptr) req = a.row_request[r];
    const int buckets = ((a.vocab - 1) >> a.bucket_shift) + 1;
    at = static_cast<long>(req) * a.lists + mine;
    const int* list_start = a.list_start + at * (buckets + 1);
    from = list_start[lo >> a.bucket_shift];
    until = list_start[((hi - 1) >> a.bucket_shift) + 1];
    at *= a.list_room;
  }
  const bool in_place = a.in == a.out && a.in_row == a.out_row;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int t0 = x.token(i);
    const uint32_t shown = x.shown(i);
    if (t0 + E <= 0 || t0 >= a.vocab || (in_place && shown == (1u << E) - 1)) continue;
    if (shown != (1u << E) - 1) {
      T* e = reinterpret_cast<T*>(&x.x[i]);
#pragma unroll
      for (int k = 0; k < E; ++k)
        if ((shown >> k & 1) == 0) e[k] = static_cast<T>(-INFINITY);
    }
    x.store(a, i);
  }
  if (!a.listed) return;
  __syncthreads();
  if (from >= until) return;
  const float rep = a.repetition != nullptr ? a.repetition[req] : 1.f;
  const float freq = a.frequency != nullptr ? a.frequency[req] : 0.f;
  const float pres = a.presence != nullptr ? a.presence[req] : 0.f;
  for (int i = from + tid - mine * share; i < until; i += share) {
    const int2 entry = a.list[at + i];
    const int t = entry.x, what = entry.y;
    if (t < lo || t >= hi) continue;
    if (a.allowed != nullptr && (a.allowed[r * a.allowed_row + (t >> 5)] >> (t & 31) & 1) == 0) continue;  // (hidden: -infinity already)
    int times = what & LG_TIMES;
    if (what & LG_DRAFT) {  // drafted nodes of this token on the way to this row
      const uint4 way = a.row_way[r];
      const int first = a.cu[req], n = min(min(a.cu[req + 1], a.rows) - first, TREE_MAX);
      for (int j = 1; j < n; ++j) {
        const uint32_t word = j < 32 ? way.x : j < 64 ? way.y : j < 96 ? way.z : way.w;
        if (word >> (j & 31) & 1) times += a.drafted[first + j] == t;
      }
    }
    const float y = lg_used(static_cast<float>(x.in[t]), times > 0 || (what & LG_PROMPT), times, rep, freq, pres, what & LG_BIAS ? a.list_bias[at + i] : 0.f);
    x.out[t] = static_cast<T>(y);
  }
}

// Where the lists of a call lie in its workspace, and how large that is.
static long lg_lists(LogitsArgs& a, void* work, int sms) {
  a.bucket_shift = 8;  // (few tokens share a bucket, and with it a counter)
  while (((a.vocab - 1) >> a.bucket_shift) + 1 > LG_BUCKETS) ++a.bucket_shift;
  const int buckets = ((a.vocab - 1) >> a.bucket_shift) + 1;
  char* at = static_cast<char*>(work);
  auto take = [&](long bytes) {
    char* was = at;
    at += (bytes + 15) / 16 * 16;
    return was;
  };
  // few requests: several CTAs count each, every one some of the tokens (by their lowest bits) for a list of its own
  a.lists = 1;
  while (a.lists < 8 && static_cast<long>(a.requests) * a.lists * 2 <= 2l * sms) a.lists *= 2;
  const long S = static_cast<long>(a.requests) * a.lists;
  // (a list has each token once, and of the vocabulary only every lists-th)
  const long listed = static_cast<long>(a.penal ? a.text + (a.cu != nullptr ? TREE_MAX : 0) : 0) + a.biases, most = (a.vocab + a.lists - 1) / a.lists;
  a.list_room = listed < most ? listed : most;
  a.row_way = reinterpret_cast<uint4*>(take(a.cu != nullptr ? a.rows * 16l : 0));
  a.row_request = reinterpret_cast<int*>(take(a.cu != nullptr ? a.rows * 4l : 0));
  a.list_start = reinterpret_cast<int*>(take(S * (buckets + 1) * 4));
  a.list = reinterpret_cast<int2*>(take(S * a.list_room * 8));
  a.list_bias = reinterpret_cast<float*>(take(a.biases > 0 ? S * a.list_room * 4 : 0));
  return at - static_cast<char*>(work);
}

// Small calls: everything in one launch, 8 tokens a thread.
static bool lg_small(const LogitsArgs& a, int sms) { return static_cast<long>((a.vocab + 7 + 2047) / 2048) * a.rows <= 8L * sms; }

template <int HASH, int THREADS>
static cudaError_t launch_count(const LogitsArgs& a, cudaStream_t s) {
  auto kern = logits_count_kernel<HASH, THREADS>;
  if (cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), 2 * HASH * 4); e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(a.requests * a.lists), dim3(THREADS), 2 * HASH * 4, s, a);
}

template <typename T>
static int launch_logits(LogitsArgs a, void* work, long work_bytes, int sms, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T), CHUNK = 4 * E * LG_THREADS;
  auto chunks_of = [&](int chunk) { return (a.vocab + E - 1 + chunk - 1) / chunk; };  // (a row may start up to E - 1 places into its first 16 bytes)
  if (a.penal || a.biases > 0) {
    if (lg_small(a, sms)) {
      a.chunks = chunks_of(2048);
      return (int)launch_pdl(logits_kernel<T, 2048>, dim3(a.chunks * a.rows), dim3(LG_THREADS), 0, s, a);
    }
    if (lg_lists(a, work, sms) > work_bytes) return (int)cudaErrorInvalidValue;
    // 64 KB of table leave room for two CTAs on an SM, 128 KB take a text of 12,000 tokens. A token's turn is a chain of looks at the table, so texts of some
    // length want more threads (256 texts of 257 to 2047: 64.4 us for the call with 1024 threads, 69.6 with 512); 512 requests with biases alone: 27.7 and 22.9.
    // The rule goes by the width of the tensor, as lengths are on the device: 256 texts of 257 to 2047 take 63 us in 2047 columns and in 32769, texts of 20 to
    // 300 take 53 in 300 columns and 58 in 32769.
    const bool wide = a.text > 1024;
    const cudaError_t e = static_cast<long>(a.text) + a.biases + TREE_MAX > 6144 ? launch_count<16384, 1024>(a, s)
                          : wide                                                   ? launch_count<8192, 1024>(a, s)
                                                                                   : launch_count<8192, 512>(a, s);
    if (e != cudaSuccess) return (int)e;
    a.listed = 1;
  }
  a.chunks = chunks_of(CHUNK);
  const long ctas = static_cast<long>(a.chunks) * a.rows;
  if (ctas > 0x7fffffffl) return (int)cudaErrorInvalidValue;
  return (int)launch_pdl(logits_row_kernel<T>, dim3(static_cast<unsigned>(ctas)), dim3(LG_THREADS), 0, s, a);
}

}  // namespace sb

// call: addresses of in, out, tokens, lengths, prompts, repetition, frequency, presence, bias ids, bias values, allowed, drafted, parents, cu (null: not there); then
// the pitches of in, out, tokens, biases and allowed (elements), rows, requests, vocabulary, tokens of a text, biases of a request, whether in and
// out are fp32 (else bf16), SMs, address
// and bytes of a workspace of the size that sb_adjust_logits_work names. in and out may be the same. Tokens outside the vocabulary (of texts, trees and biases) count for nothing. With trees, row r is
// node r - cu[b] of tree b; rows behind cu[requests] are left as they are.
extern "C" int sb_adjust_logits(const void* call, cudaStream_t s) {
  const long long* x = static_cast<const long long*>(call);
  auto ints = [&](int i) { return reinterpret_cast<const int*>(x[i]); };
  auto floats = [&](int i) { return reinterpret_cast<const float*>(x[i]); };
  sb::LogitsArgs a = {};
  a.in = reinterpret_cast<const void*>(x[0]);
  a.out = reinterpret_cast<void*>(x[1]);
  a.tokens = ints(2); a.lengths = ints(3); a.prompts = ints(4);
  a.repetition = floats(5); a.frequency = floats(6); a.presence = floats(7);
  a.bias_ids = ints(8); a.bias_values = floats(9);
  a.allowed = ints(10);
  a.drafted = ints(11); a.parents = ints(12); a.cu = ints(13);
  a.in_row = x[14]; a.out_row = x[15]; a.tokens_row = x[16]; a.bias_row = x[17]; a.allowed_row = x[18];
  a.rows = x[19]; a.requests = x[20]; a.vocab = x[21]; a.text = x[22]; a.biases = x[23];
  if (a.rows <= 0 || a.vocab <= 0) return 0;
  a.penal = a.repetition != nullptr || a.frequency != nullptr || a.presence != nullptr;
  const int sms = static_cast<int>(x[25]);
  void* work = reinterpret_cast<void*>(x[26]);
  return x[24] ? sb::launch_logits<float>(a, work, x[27], sms, s) : sb::launch_logits<__nv_bfloat16>(a, work, x[27], sms, s);
}

// Bytes of workspace of a call with so many rows, requests, tokens of vocabulary and of a text (0: no penalties) and biases; 0: it needs none.
extern "C" int sb_adjust_logits_work(int rows, int requests, int vocab, int text, int biases, int penal, int tree, int sms, long* bytes) {
  static const int some = 0;
  sb::LogitsArgs a = {};
  a.rows = rows;
  a.requests = requests;
  a.vocab = vocab;
  a.text = text;
  a.biases = biases;
  a.penal = penal;
  a.cu = tree ? &some : nullptr;
  *bytes = (penal || biases > 0) && rows > 0 && vocab > 0 && !sb::lg_small(a, sms) ? sb::lg_lists(a, nullptr, sms) : 0;
  return 0;
}
