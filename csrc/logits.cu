// Logits before sampling: penalties for tokens of the text, biases, and the mask of a grammar, in one pass (sm_100a).
//
//   x = logits[r, t];  c = times that t was answered with (or drafted on the way to node r), seen = c > 0 or t is in the prompt
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - c * frequency - (c > 0) * presence + sum of the biases of t;   x = -inf where the mask's bit of t is 0
//
// Nearly all logits of a row are only copied or masked. So calls of some size take two launches: `logits_mask_kernel` copies and masks at the rate of
// memory, and `logits_used_kernel` works out the few tokens that were used or have a bias. For that a CTA counts a request's text into a table
// of 16384 tokens of the vocabulary in shared memory, and each token's first taker works it out for all rows of the request: a request needs
// no table of the vocabulary's size that would have to be kept, cleared and read, only its text. Small calls take one launch,
// `logits_kernel`, that keeps a chunk of a row in registers while it counts.
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
  int parts, slices;      // of the vocabulary; CTAs that share the rows of a tree
  int penal;
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

// Adds the text of a request to a table of the tokens [base, base + size): LG_PROMPT, or 1 for every other time.
enum : int { LG_PROMPT = 1 << 30, LG_BIAS = 1 << 29, LG_DRAFT = 1 << 28, LG_TAKEN = 1 << 27 };
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
        if (c != 0) v = lg_used(v, (c & ~LG_BIAS) != 0, c & (LG_TAKEN - 1), rep, freq, pres, any_bias ? bias[at + q + k] : 0.f);
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

constexpr int LG_PART = 16384;       // tokens of a table
constexpr int LG_USED_THREADS = 512;

template <typename T>
__global__ void __launch_bounds__(LG_USED_THREADS)
logits_used_kernel(const __grid_constant__ LogitsArgs a) {
  extern __shared__ __align__(16) int count[];
  __shared__ int tree_p[TREE_MAX], tree_t[TREE_MAX];
  __shared__ __align__(16) uint4 ways[TREE_MAX];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int part = blockIdx.x % a.parts, slice = blockIdx.x / a.parts % a.slices, req = blockIdx.x / (a.parts * a.slices);
  int first = req, until = req + 1, n = 0;
  if (a.cu != nullptr) {
    first = a.cu[req];
    until = min(a.cu[req + 1], a.rows);
    n = min(until - first, TREE_MAX);
  }
  if (first < 0 || first + slice >= until) return;
  const float rep = a.repetition != nullptr ? a.repetition[req] : 1.f;
  const float freq = a.frequency != nullptr ? a.frequency[req] : 0.f;
  const float pres = a.presence != nullptr ? a.presence[req] : 0.f;
  const bool counts = a.penal && (rep != 1.f || freq != 0.f || pres != 0.f);
  const int K = a.biases;
  if (!counts && K == 0) return;
  const int base = part * LG_PART, size = min(LG_PART, a.vocab - base);
  const int* ids = a.bias_ids + req * a.bias_row;
  const float* values = a.bias_values + req * a.bias_row;
  auto place = [&](int t) { return t >= base && t - base < size ? t - base : -1; };
  for (int i = tid; i < LG_PART / 4; i += LG_USED_THREADS) reinterpret_cast<int4*>(count)[i] = make_int4(0, 0, 0, 0);
  for (int i = tid; counts && i < n; i += LG_USED_THREADS) {
    tree_p[i] = a.parents[first + i];
    tree_t[i] = a.drafted[first + i];
  }
  __syncthreads();
  // ---- what there is of each token
  int again = 0;
  if (counts) {
    const int prompt = a.prompts != nullptr ? a.prompts[req] : 0;
    lg_text(a, req, LG_USED_THREADS, [&](int i, int t) {
      if (const int at = place(t); at >= 0) {
        if (i < prompt) atomicOr(&count[at], LG_PROMPT);
        else atomicAdd(&count[at], 1);
      }
    });
    if (tid < n) {
      uint32_t set[4];
      tree_way_up([&](int j) { return tree_p[j]; }, tid, set);
      ways[tid] = make_uint4(set[0] & ~1u, set[1], set[2], set[3]);  // (the root is the text's last token)
      if (const int at = place(tree_t[tid]); tid > 0 && at >= 0) atomicOr(&count[at], LG_DRAFT);
    }
  }
  for (int i = tid; i < K; i += LG_USED_THREADS)
    if (const int at = place(ids[i]); at >= 0) again |= (atomicOr(&count[at], LG_BIAS) & LG_BIAS) != 0;  // listed twice
  again = __syncthreads_or(again);
  // ---- the first to take a token works it out for this CTA's rows. entry: of the list of biases, or -1
  auto take = [&](int t, int entry) {
    const int at = place(t);
    if (at < 0) return;
    if (count[at] & LG_TAKEN) return;
    const int c = atomicOr(&count[at], LG_TAKEN);
    if (c & LG_TAKEN) return;
    float bias = 0.f;
    if (c & LG_BIAS) {
      if (entry >= 0 && !again) {
        bias = values[entry];
      } else {
        for (int j = 0; j < K; ++j)
          if (ids[j] == t) bias += values[j];
      }
    }
    uint32_t nodes[4] = {0, 0, 0, 0};  // that stand for this token
    if (c & LG_DRAFT)
      for (int j = 1; j < n; ++j)
        if (tree_t[j] == t) {
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (j >> 5 == w) nodes[w] |= 1u << (j & 31);
        }
    const int times0 = c & (LG_TAKEN - 1);
    constexpr int FLY = 4;  // rows whose reads are under way together
    for (int r0 = first + slice; r0 < until; r0 += FLY * a.slices) {
      T v[FLY];
      uint32_t word[FLY];
#pragma unroll
      for (int x = 0; x < FLY; ++x) {
        const int r = r0 + x * a.slices;
        word[x] = 0xffffffffu;
        if (r < until) {
          v[x] = reinterpret_cast<const T*>(a.in)[r * a.in_row + t];
          if (a.allowed != nullptr) word[x] = static_cast<uint32_t>(a.allowed[r * a.allowed_row + (t >> 5)]);
        }
      }
#pragma unroll
      for (int x = 0; x < FLY; ++x) {
        const int r = r0 + x * a.slices;
        if (r >= until) break;
        int times = times0;
        if ((c & LG_DRAFT) && r - first < n) {
          const uint4 w = ways[r - first];
          times += __popc(w.x & nodes[0]) + __popc(w.y & nodes[1]) + __popc(w.z & nodes[2]) + __popc(w.w & nodes[3]);
        }
        if ((word[x] >> (t & 31) & 1) == 0) continue;  // (-infinity already)
        const float y = lg_used(static_cast<float>(v[x]), times > 0 || (c & LG_PROMPT), times, rep, freq, pres, bias);
        reinterpret_cast<T*>(a.out)[r * a.out_row + t] = static_cast<T>(y);
      }
    }
  };
  for (int i = tid; i < K; i += LG_USED_THREADS) take(ids[i], i);
  if (counts) {
    if (tid > 0 && tid < n) take(tree_t[tid], -1);
    lg_text(a, req, LG_USED_THREADS, [&](int, int t) { take(t, -1); });
  }
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
  }
  if (!used) return 0;
  a.parts = (a.vocab + LG_PART - 1) / LG_PART;
  // CTAs that share the rows of a tree: each counts the text for itself
  const long ctas = static_cast<long>(a.parts) * a.requests;
  a.slices = a.cu == nullptr ? 1 : static_cast<int>(ctas >= 6L * sms ? 1 : (6L * sms + ctas - 1) / ctas);
  if (a.slices > 8) a.slices = 8;
  if (ctas * a.slices > 0x7fffffffl) return (int)cudaErrorInvalidValue;
  if (cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(logits_used_kernel<T>), LG_PART * 4); e != cudaSuccess) return (int)e;
  return (int)launch_pdl(logits_used_kernel<T>, dim3(static_cast<unsigned>(ctas * a.slices)), dim3(LG_USED_THREADS), LG_PART * 4, s, a);
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
