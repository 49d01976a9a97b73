// Logits before sampling: penalties for tokens of the text, biases, and the mask of a grammar, in one pass (sm_100a).
//
//   x = logits[r, t];  c = times that t was answered with (or drafted on the way to node r), seen = c > 0 or t is in the prompt
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - c * frequency - (c > 0) * presence + sum of the biases of t;   x = -inf where the mask's bit of t is 0
//
// Nearly all logits of a row are only copied or masked. So calls of some size take two launches: `logits_mask_kernel` copies and masks at the rate of
// memory, and `logits_used_kernel` works out the few tokens that were used or have a bias. For that a CTA counts a request's text in a
// hash table in shared memory, whose places then are the work list for all rows of the request: a request needs no table of the
// vocabulary's size that would have to be kept, cleared and read, only its text. Small calls take one launch, `logits_kernel`, that
// keeps a chunk of a row in registers while it counts.
// Biases of a token are added up in list order by one thread: nothing depends on an order of arrival. Logits that the mask hides are not read.
// Everything is worked out in fp32 and rounded once. What bounds it: reading and writing the logits, 16 bytes a thread and access; a row that
// does not start on such a boundary is cut at the boundaries all the same, and its two ends go element by element.
#include "token_tree.cuh"

namespace sb {

constexpr int LG_THREADS = 256;

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
  int slices;             // CTAs that share the rows of a tree
  int penal;
  int behind_mask;        // the launch in front of this one is logits_mask_kernel
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

// What there is of a token: in the prompt, has a bias, was drafted, and how many times it was answered with. lg_text: each token of a request's text.
enum : int { LG_PROMPT = 1 << 30, LG_BIAS = 1 << 29, LG_DRAFT = 1 << 28 };
template <typename F>
__device__ __forceinline__ void lg_text(const LogitsArgs& a, int req, int threads, const F& each) {
  const int* text = a.tokens + req * a.tokens_row;
  const int len = max(min(a.lengths[req], a.text), 0);
  int from = 0;
  if ((reinterpret_cast<uintptr_t>(text) & 15) == 0) {
    from = len & ~3;
    for (int i = 4 * threadIdx.x; i < from; i += 4 * threads) {
      const int4 t = *reinterpret_cast<const int4*>(text + i);
      each(i, t.x);
      each(i + 1, t.y);
      each(i + 2, t.z);
      each(i + 3, t.w);
    }
  }
  for (int i = from + threadIdx.x; i < len; i += threads) each(i, text[i]);
}

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
    n = min(min(a.cu[req + 1], a.rows) - first, TREE_MAX);
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
    lg_text(a, req, LG_THREADS, [&](int i, int t) {
      if (const int at = place(t); at >= 0) {
        if (i < prompt) atomicOr(&count[at], LG_PROMPT);
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
  int any_bias = 0, again = 0;
  const int K = a.biases;
  const int* ids = a.bias_ids + req * a.bias_row;
  const float* values = a.bias_values + req * a.bias_row;
  for (int i = tid; i < K; i += LG_THREADS)
    if (const int at = place(ids[i]); at >= 0) {
      again |= (atomicOr(&count[at], LG_BIAS) & LG_BIAS) != 0;  // listed twice
      any_bias = 1;
    }
  again = __syncthreads_or(again);
  any_bias = __syncthreads_or(any_bias);
  if (any_bias) {
    for (int i = tid; i < K; i += LG_THREADS)
      if (const int id = ids[i], at = place(id); at >= 0) {
        float sum = values[i];
        if (again) {  // all entries of a token add up the same: which one is written does not matter
          sum = 0.f;
          for (int j = 0; j < K; ++j)
            if (ids[j] == id) sum += values[j];
        }
        bias[at] = sum;
      }
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
        if (c != 0) v = lg_used(v, (c & ~LG_BIAS) != 0, c & (LG_DRAFT - 1), rep, freq, pres, any_bias ? bias[at + q + k] : 0.f);
        if ((shown >> (q + k) & 1) == 0) v = -INFINITY;
        e[q + k] = static_cast<T>(v);
      }
    }
    x.store(a, i);
  }
}

// ---------------------------------------------------------------- two launches: copy and mask; then the tokens that were used or have a bias
template <typename T>
__global__ void __launch_bounds__(LG_THREADS)
logits_mask_kernel(const __grid_constant__ LogitsArgs a) {
  constexpr int NV = 4, E = 16 / sizeof(T);
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.x / a.chunks, chunk = blockIdx.x - r * a.chunks;
  if (a.cu != nullptr && (r < a.cu[0] || r >= a.cu[a.requests])) return;  // not a row of a tree: left as it is
  Pieces<T, NV> x;
  x.load(a, r, chunk * (NV * E * LG_THREADS));
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
}

// The tokens of a request that were used, drafted or have a bias, worked out for every `slices`-th row of the request. They are counted in a hash table
// of HASH places in shared memory (linear probing, at most three quarters full), whose places then are the work list; a longer text
// is counted in a table of 2 HASH tokens of the vocabulary at a time instead.
template <typename T, int HASH>
__global__ void __launch_bounds__(HASH / 16, HASH == 8192 ? 2 : 1)
logits_used_kernel(const __grid_constant__ LogitsArgs a) {
  constexpr int THREADS = HASH / 16;
  extern __shared__ __align__(16) int tables[];
  int* keys = tables;          // [HASH] token, -1: empty
  int* hashed = tables + HASH;  // [HASH] what there is of it
  uint16_t* list = reinterpret_cast<uint16_t*>(tables + 2 * HASH);  // occupied places
  __shared__ int listed;
  __shared__ int tree_p[TREE_MAX], tree_t[TREE_MAX];
  __shared__ __align__(16) uint4 ways[TREE_MAX];
  // What is counted was there before the launch in front of this one, which has waited for it: only the rows have to be masked first.
  if (!a.behind_mask) pdl_wait();
  const int tid = threadIdx.x;
  const int slice = blockIdx.x % a.slices, req = blockIdx.x / a.slices;
  int first = req, until = req + 1, n = 0;
  if (a.cu != nullptr) {
    first = a.cu[req];
    until = min(a.cu[req + 1], a.rows);
    n = min(until - first, TREE_MAX);
  }
  const float rep = a.repetition != nullptr ? a.repetition[req] : 1.f;
  const float freq = a.frequency != nullptr ? a.frequency[req] : 0.f;
  const float pres = a.presence != nullptr ? a.presence[req] : 0.f;
  const bool counts = a.penal && (rep != 1.f || freq != 0.f || pres != 0.f);
  const int K = a.biases;
  if (first < 0 || first + slice >= until || (!counts && K == 0)) {
    pdl_wait();  // (every launch of a chain waits for the one in front of it)
    return;
  }
  const int* ids = a.bias_ids + req * a.bias_row;
  const float* values = a.bias_values + req * a.bias_row;
  const int len = counts ? max(min(a.lengths[req], a.text), 0) : 0;
  const int prompt = counts && a.prompts != nullptr ? a.prompts[req] : 0;
  if (tid == 0) listed = 0;
  const bool direct = static_cast<long>(len) + K + n > HASH / 4 * 3;
  for (int i = tid; counts && i < n; i += THREADS) {
    tree_p[i] = a.parents[first + i];
    tree_t[i] = a.drafted[first + i];
  }
  const int passes = direct ? (a.vocab + 2 * HASH - 1) / (2 * HASH) : 1;
  for (int pass = 0; pass < passes; ++pass) {
    const int base = pass * 2 * HASH;
    const int4 empty = direct ? make_int4(0, 0, 0, 0) : make_int4(-1, -1, -1, -1);
    for (int i = tid; i < HASH / 4; i += THREADS) {
      reinterpret_cast<int4*>(keys)[i] = empty;
      reinterpret_cast<int4*>(hashed)[i] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
    // ---- what there is of each token
    auto place = [&](int t) -> int* {
      if (static_cast<unsigned>(t) >= static_cast<unsigned>(a.vocab)) return nullptr;
      if (direct) return t >= base && t - base < 2 * HASH ? tables + (t - base) : nullptr;
      unsigned at = (static_cast<unsigned>(t) * 2654435761u) >> 16;  // Knuth's multiplicative hashing
      while (true) {
        at &= HASH - 1;
        const int was = atomicCAS(&keys[at], -1, t);
        if (was == -1 || was == t) return &hashed[at];
        ++at;
      }
    };
    if (counts) {
      lg_text(a, req, THREADS, [&](int i, int t) {
        if (int* at = place(t); at != nullptr) {
          if (i < prompt) atomicOr(at, LG_PROMPT);
          else atomicAdd(at, 1);
        }
      });
      if (tid < n) {
        if (pass == 0) {
          uint32_t set[4];
          tree_way_up([&](int j) { return tree_p[j]; }, tid, set);
          ways[tid] = make_uint4(set[0] & ~1u, set[1], set[2], set[3]);  // (the root is the text's last token)
        }
        if (tid > 0)
          if (int* at = place(tree_t[tid]); at != nullptr) atomicOr(at, LG_DRAFT);
      }
    }
    // biases: the first of a token's entries to come works the token out. again: a token is listed twice. mine: entries, one bit each
    const bool marks = K <= 32 * THREADS;
    uint32_t mine = 0;
    int again = 0;
    for (int i = tid, x = 0; i < K; i += THREADS, ++x)
      if (int* at = place(ids[i]); at != nullptr) {
        const bool came = (atomicOr(at, LG_BIAS) & LG_BIAS) == 0;
        if (came && marks) mine |= 1u << x;
        again |= !came;
      }
    again = __syncthreads_or(again);
    if (pass == 0) {
      if (a.behind_mask) pdl_wait();
      pdl_launch_dependents();
    }
    // ---- each token's logits
    constexpr int FLY = 4;  // logits whose reads are under way together
    const int step = a.slices, rows = (until - first - slice + step - 1) / step;  // this CTA's rows: first + slice + x step
    // c 0: nothing to do
    auto work = [&](const int (&t)[FLY], const int (&c)[FLY], const int (&r)[FLY], float bias) {
      T v[FLY];
      uint32_t word[FLY];
#pragma unroll
      for (int x = 0; x < FLY; ++x) {
        word[x] = c[x] != 0 ? 0xffffffffu : 0u;
        if (c[x] == 0) continue;
        v[x] = reinterpret_cast<const T*>(a.in)[r[x] * a.in_row + t[x]];
        if (a.allowed != nullptr) word[x] = static_cast<uint32_t>(a.allowed[r[x] * a.allowed_row + (t[x] >> 5)]);
      }
#pragma unroll
      for (int x = 0; x < FLY; ++x) {
        if ((word[x] >> (t[x] & 31) & 1) == 0) continue;  // (hidden: -infinity already)
        int times = c[x] & (LG_DRAFT - 1);
        if ((c[x] & LG_DRAFT) && r[x] - first < n) {
          const uint32_t* way = reinterpret_cast<const uint32_t*>(&ways[r[x] - first]);
          for (int j = 1; j < n; ++j) times += tree_t[j] == t[x] && (way[j >> 5] >> (j & 31) & 1);
        }
        const float y = lg_used(static_cast<float>(v[x]), times > 0 || (c[x] & LG_PROMPT), times, rep, freq, pres, bias);
        reinterpret_cast<T*>(a.out)[r[x] * a.out_row + t[x]] = static_cast<T>(y);
      }
    };
    if (!direct) {
      // the occupied places side by side; (place, row) pairs are dealt out evenly
      for (int p0 = 0; p0 < HASH; p0 += THREADS) {
        const int c = hashed[p0 + tid];
        const bool some = c != 0 && (c & LG_BIAS) == 0;
        const uint32_t all = __ballot_sync(0xffffffffu, some);
        int at = 0;
        if ((tid & 31) == 0 && all != 0) at = atomicAdd(&listed, __popc(all));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(all & ((1u << (tid & 31)) - 1));
        if (some) list[at] = static_cast<uint16_t>(p0 + tid);
      }
      __syncthreads();
      const int m = listed;
      for (int p0 = tid; p0 < m * rows; p0 += FLY * THREADS) {
        int t[FLY], c[FLY], r[FLY];
#pragma unroll
        for (int x = 0; x < FLY; ++x) {
          const int p = p0 + x * THREADS;
          const bool some = p < m * rows;
          const int row = some ? p / m : 0, at = some ? list[p - row * m] : 0;
          t[x] = some ? keys[at] : 0;
          c[x] = some ? hashed[at] : 0;
          r[x] = first + slice + row * step;
        }
        work(t, c, r, 0.f);
      }
    } else {
      for (int p0 = tid; p0 < 2 * HASH; p0 += FLY * THREADS) {
        int t[FLY], c[FLY];
#pragma unroll
        for (int x = 0; x < FLY; ++x) {
          const int at = p0 + x * THREADS;
          t[x] = base + at;
          c[x] = tables[at];
          if (c[x] & LG_BIAS) c[x] = 0;
        }
        if ((c[0] | c[1] | c[2] | c[3]) != 0)
          for (int r0 = first + slice; r0 < until; r0 += step) {
            const int r[FLY] = {r0, r0, r0, r0};
            work(t, c, r, 0.f);
          }
      }
    }
    for (int i = tid, x = 0; i < K; i += THREADS, ++x) {
      const int id = ids[i];
      if (marks && (mine >> x & 1) == 0) continue;
      const int* at = place(id);
      if (at == nullptr) continue;
      bool leads = true;
      for (int j = 0; !marks && leads && j < i; ++j) leads = ids[j] != id;
      if (!leads) continue;
      float bias = values[i];
      if (again) {
        bias = 0.f;
        for (int j = 0; j < K; ++j)
          if (ids[j] == id) bias += values[j];
      }
      const int what = *at, t[FLY] = {id, id, id, id};
      for (int r0 = first + slice; r0 < until; r0 += FLY * step) {
        int c[FLY], r[FLY];
#pragma unroll
        for (int y = 0; y < FLY; ++y) {
          r[y] = r0 + y * step;
          c[y] = r[y] < until ? what : 0;
        }
        work(t, c, r, bias);
      }
    }
    if (pass + 1 < passes) __syncthreads();
  }
}

template <typename T, int HASH>
static int launch_used(LogitsArgs a, int sms, cudaStream_t s) {
  // CTAs that share the rows of a tree: each counts the text for itself
  a.slices = a.cu == nullptr ? 1 : static_cast<int>(a.requests >= 2l * sms ? 1 : 2l * sms / a.requests);
  if (a.slices > 8) a.slices = 8;
  if (static_cast<long>(a.requests) * a.slices > 0x7fffffffl) return (int)cudaErrorInvalidValue;
  auto kern = logits_used_kernel<T, HASH>;
  constexpr int bytes = 2 * HASH * 4 + HASH / 4 * 3 * 2;
  if (cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), bytes); e != cudaSuccess) return (int)e;
  return (int)launch_pdl(kern, dim3(a.requests * a.slices), dim3(HASH / 16), bytes, s, a);
}

template <typename T>
static int launch_logits(LogitsArgs a, int sms, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T), SMALL = 2048, LARGE = 4 * E * LG_THREADS;
  auto chunks_of = [&](int chunk) { return (a.vocab + E - 1 + chunk - 1) / chunk; };  // (a row may start up to E - 1 places into its first 16 bytes)
  const bool used = a.penal || a.biases > 0;
  if (used && static_cast<long>(chunks_of(SMALL)) * a.rows <= 8L * sms) {
    a.chunks = chunks_of(SMALL);
    return (int)launch_pdl(logits_kernel<T, SMALL>, dim3(a.chunks * a.rows), dim3(LG_THREADS), 0, s, a);
  }
  if (a.allowed != nullptr || a.in != a.out || a.in_row != a.out_row) {
    a.chunks = chunks_of(LARGE);
    const long ctas = static_cast<long>(a.chunks) * a.rows;
    if (ctas > 0x7fffffffl) return (int)cudaErrorInvalidValue;
    if (cudaError_t e = launch_pdl(logits_mask_kernel<T>, dim3(static_cast<unsigned>(ctas)), dim3(LG_THREADS), 0, s, a); e != cudaSuccess) return (int)e;
    a.behind_mask = 1;
  }
  if (!used) return 0;
  // 64 KB of table leave room for three CTAs on an SM, 128 KB take a text of 12,000 tokens
  return static_cast<long>(a.text) + a.biases + TREE_MAX <= 6144 ? launch_used<T, 8192>(a, sms, s) : launch_used<T, 16384>(a, sms, s);
}

}  // namespace sb

// call: addresses of in, out, tokens, lengths, prompts, repetition, frequency, presence, bias ids, bias values, allowed, drafted, parents, cu (null: not there); then
// the pitches of in, out, tokens, biases and allowed (elements), rows, requests, vocabulary, tokens of a text, biases of a request, whether in and
// out are fp32 (else bf16), SMs. in and out may be the same. Tokens outside the vocabulary (of texts, trees and biases) count for nothing. With trees, row r is
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
  return x[24] ? sb::launch_logits<float>(a, sms, s) : sb::launch_logits<__nv_bfloat16>(a, sms, s);
}
