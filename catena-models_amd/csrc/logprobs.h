// Log probabilities of given tokens, entropy and the most likely tokens of rows of
// logits.
#pragma once

#include "layers.h"

namespace cq35 {

constexpr int kLogprobsMostTop = 32;
constexpr int kLogprobsMostGiven = 1024;

struct LogprobArgs {
  const void* logits;
  int64_t stride, rows;
  int vocab;
  const int64_t* tokens;
  int given, top;
  float *logprobs, *entropy;
  int64_t* top_tokens;
  float* top_logprobs;
};

__device__ __forceinline__ float widened(uint16_t x) { return bf2f(x); }
__device__ __forceinline__ float widened(float x) { return x; }

// Larger for larger logits (NaN above infinity, -0 as 0), among equal ones for lower indices;
// never 0 and never all ones.
__device__ __forceinline__ uint64_t logit_key(float x, int index) {
  const uint32_t b = fbits(x + 0.0f);
  const uint32_t order = x != x ? 0xfffffffeu : b >> 31 ? ~b : b | 0x80000000u;
  return (uint64_t)order << 32 | (0xffffffffu - (uint32_t)index);
}

constexpr int kLogprobThreads = 256;

// A block a row.
template <typename T>
__global__ __launch_bounds__(kLogprobThreads) void k_logprobs(LogprobArgs a) {
  __shared__ float part[3][kLogprobThreads];
  __shared__ uint64_t best[kLogprobThreads / 64];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.logits + row * a.stride;
  float m = -__builtin_inff();
  for (int i = tid; i < a.vocab; i += kLogprobThreads) m = fmaxf(m, widened(x[i]));
  part[0][tid] = m;
  __syncthreads();
  for (int i = 0; i < kLogprobThreads; ++i) m = fmaxf(m, part[0][i]);
  float s = 0.0f, t = 0.0f;
  const float from = m > -__builtin_inff() ? m : 0.0f;
  for (int i = tid; i < a.vocab; i += kLogprobThreads) {
    const float d = widened(x[i]) - from, e = __builtin_amdgcn_exp2f(d * 1.44269504f);
    s += e, t += e * fmaxf(d, -200.0f);
  }
  part[1][tid] = s, part[2][tid] = t;
  __syncthreads();
  s = t = 0.0f;
  for (int i = 0; i < kLogprobThreads; ++i) s += part[1][i], t += part[2][i];
  const float log_s = logf(s);
  if (tid == 0) a.entropy[row] = log_s - t / s;
  for (int i = tid; i < a.given; i += kLogprobThreads) {
    const int64_t token = a.tokens[row * a.given + i];
    a.logprobs[row * a.given + i] = token >= 0 && token < a.vocab ? (widened(x[token]) - m) - log_s : __builtin_nanf("");
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t mine = 0;
    for (int i = tid; i < a.vocab; i += kLogprobThreads) {
      const uint64_t key = logit_key(widened(x[i]), i);
      if (key < last && key > mine) mine = key;
    }
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)mine, d, 64);
      mine = o > mine ? o : mine;
    }
    if ((tid & 63) == 0) best[tid >> 6] = mine;
    __syncthreads();
    for (int w = 0; w < kLogprobThreads / 64; ++w) mine = best[w] > mine ? best[w] : mine;
    __syncthreads();
    last = mine;
    if (tid == 0) {
      const int64_t token = 0xffffffffu - (uint32_t)mine;
      a.top_tokens[row * a.top + k] = token;
      a.top_logprobs[row * a.top + k] = (widened(x[token]) - m) - log_s;
    }
  }
}

}  // namespace cq35
