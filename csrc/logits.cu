// Logits before sampling: penalties for tokens of the text, biases, and the mask of a grammar, in one pass (sm_100a).
//
//   x = logits[r, t];  c = times that t was answered with (or drafted on the way to node r), seen = c > 0 or t is in the prompt
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - c * frequency - (c > 0) * presence + sum of the biases of t;   x = -inf where the mask's bit of t is 0
//
// One CTA per row and chunk of LG_CHUNK tokens. Its logits are loaded first and wait in registers while the CTA counts: every thread
// reads tokens of the request's text and adds those that fall into the chunk to a table in shared memory (bit 30: in the prompt),
// so a request needs no table of the vocabulary's size that would have to be kept, cleared and read, only its text. The
// biases of a token are added up by one thread in list order: the result does not depend on any order of arrival.
// Everything is worked out in fp32 and rounded once. What bounds it: reading and writing the logits, 8 bytes a token in fp32.
#include "token_tree.cuh"

namespace sb {

constexpr int LG_THREADS = 256;
constexpr int LG_CHUNK = 4096;

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
};

template <typename T>
__device__ __forceinline__ float lg_load(const T* p) {
  return static_cast<float>(*p);
}

template <typename T>
__global__ void __launch_bounds__(LG_THREADS)
logits_kernel(const __grid_constant__ LogitsArgs a) {
  __shared__ int count[LG_CHUNK];
  __shared__ float bias[LG_CHUNK];
  __shared__ int tree_p[TREE_MAX], tree_t[TREE_MAX];
  __shared__ int found;
  pdl_wait();
  pdl_launch_dependents();
  const int chunks = (a.vocab + LG_CHUNK - 1) / LG_CHUNK;
  const int r = blockIdx.x / chunks, tid = threadIdx.x;
  const int c0 = (blockIdx.x - r * chunks) * LG_CHUNK, cn = min(LG_CHUNK, a.vocab - c0);
  const T* in = reinterpret_cast<const T*>(a.in) + r * a.in_row + c0;
  T* out = reinterpret_cast<T*>(a.out) + r * a.out_row + c0;
  float x[LG_CHUNK / LG_THREADS];
#pragma unroll
  for (int i = 0; i < LG_CHUNK / LG_THREADS; ++i) x[i] = i * LG_THREADS + tid < cn ? lg_load(in + i * LG_THREADS + tid) : 0.f;
  // ---- whose row it is
  int req = r;
  if (a.cu != nullptr) {
    if (tid == 0) found = -1;
    __syncthreads();
    for (int b = tid; b < a.requests; b += LG_THREADS)
      if (max(a.cu[b], 0) <= r && r < a.cu[b + 1]) found = b;
    __syncthreads();
    req = found;
    if (req < 0) return;  // behind the last tree: left as it is
  }
  const float rep = a.repetition != nullptr ? a.repetition[req] : 1.f;
  const float freq = a.frequency != nullptr ? a.frequency[req] : 0.f;
  const float pres = a.presence != nullptr ? a.presence[req] : 0.f;
  const bool counts = rep != 1.f || freq != 0.f || pres != 0.f;
  // ---- tables of this chunk
  for (int i = tid; i < LG_CHUNK; i += LG_THREADS) {
    count[i] = 0;
    bias[i] = 0.f;
  }
  __syncthreads();
  if (counts) {
    const int* text = a.tokens + req * a.tokens_row;
    const int len = min(a.lengths[req], a.text), prompt = a.prompts != nullptr ? a.prompts[req] : 0;
    for (int i = tid; i < len; i += LG_THREADS) {
      const unsigned at = static_cast<unsigned>(text[i] - c0);
      if (at < static_cast<unsigned>(cn)) {
        if (i < prompt) atomicOr(&count[at], 1 << 30);
        else atomicAdd(&count[at], 1);
      }
    }
    if (a.cu != nullptr) {
      const int first = a.cu[req], n = min(min(a.cu[req + 1], a.rows) - first, TREE_MAX);
      for (int i = tid; i < n; i += LG_THREADS) {
        tree_p[i] = a.parents[first + i];
        tree_t[i] = a.drafted[first + i];
      }
      __syncthreads();
      uint32_t way[4];
      if (r - first < n) {
        tree_way_up([&](int j) { return tree_p[j]; }, r - first, way);
        if (tid > 0 && tid < n) {
          uint32_t word = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (tid >> 5 == w) word = way[w];
          const unsigned at = static_cast<unsigned>(tree_t[tid] - c0);
          if ((word >> (tid & 31) & 1) && at < static_cast<unsigned>(cn)) atomicAdd(&count[at], 1);
        }
      }
    }
  }
  int any_bias = 0;
  if (a.biases > 0) {
    const int* ids = a.bias_ids + req * a.bias_row;
    const float* values = a.bias_values + req * a.bias_row;
    for (int i = tid; i < a.biases; i += LG_THREADS) {
      const int id = ids[i];
      if (id < c0 || id >= c0 + cn) continue;
      any_bias = 1;
      bool first = true;
      for (int j = 0; j < i && first; ++j) first = ids[j] != id;
      if (!first) continue;
      float sum = values[i];
      for (int j = i + 1; j < a.biases; ++j)
        if (ids[j] == id) sum += values[j];
      bias[id - c0] = sum;
    }
  }
  any_bias = __syncthreads_or(any_bias);
  // ---- the row
  const int* allowed = a.allowed != nullptr ? a.allowed + r * a.allowed_row : nullptr;
#pragma unroll
  for (int i = 0; i < LG_CHUNK / LG_THREADS; ++i) {
    const int at = i * LG_THREADS + tid;
    if (at >= cn) break;
    float v = x[i];
    const int c = count[at];
    if (c != 0) {
      v = v > 0.f ? v / rep : v * rep;
      const int times = c & ((1 << 30) - 1);
      if (times > 0) v = v - freq * static_cast<float>(times) - pres;
    }
    if (any_bias) v += bias[at];
    if (allowed != nullptr && (allowed[(c0 + at) >> 5] >> ((c0 + at) & 31) & 1) == 0) v = -INFINITY;
    out[at] = static_cast<T>(v);
  }
}

}  // namespace sb

// call: addresses of in, out, tokens, lengths, prompts, repetition, frequency, presence, bias ids, bias values, allowed, drafted, parents, cu (null: not there); then
// the pitches of in, out, tokens, biases and allowed (elements), rows, requests, vocabulary, tokens of a text, biases of a request, whether in and
// out are fp32 (else bf16). in and out may be the same. Tokens outside the vocabulary (of texts, trees and biases) count for nothing. With trees, row r is
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
  const dim3 block(sb::LG_THREADS);
  const long ctas = (static_cast<long>(a.vocab) + sb::LG_CHUNK - 1) / sb::LG_CHUNK * a.rows;
  if (ctas > 0x7fffffffl) return (int)cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(ctas));
  return (int)(x[24] ? sb::launch_pdl(sb::logits_kernel<float>, grid, block, 0, s, a) : sb::launch_pdl(sb::logits_kernel<__nv_bfloat16>, grid, block, 0, s, a));
}
