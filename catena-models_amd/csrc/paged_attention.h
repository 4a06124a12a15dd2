// Attention of new tokens over a paged KV cache.
#pragma once

#include "mfma.h"
#include "paged_index.h"

namespace cq35 {

struct AttendArgs {
  const uint16_t *q, *gate;  // gate: null without
  uint16_t* out;
  int64_t q_row, q_head, gate_row, gate_head, out_row, out_head;
  const uint16_t *keys, *values;
  int64_t pages, page_stride, row_stride, head_stride;
  int shift;
  const int32_t* table;
  int64_t table_stride, width;
  const int32_t *row_start, *lengths;
  int requests;
  int64_t rows;
  int q_heads, kv_heads, group;
  float scale;
};

// One block per (row, query head); each wave every fourth key.
constexpr int kSimpleThreads = 256;
template <int HD>
__global__ __launch_bounds__(kSimpleThreads) void k_paged_simple(AttendArgs a) {
  constexpr int E = HD / 64;
  __shared__ float ms[4], ds[4], os[4][HD];
  const int64_t t = blockIdx.x;
  const int head = blockIdx.y, kvh = head / a.group, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (a.row_start[0] > t) return;
  const int r = request_of(a.row_start, a.requests, t);
  const int64_t begin = a.row_start[r], end = a.row_start[r + 1];
  if (t >= end) return;
  const int64_t length = max((int64_t)0, min((int64_t)a.lengths[r], a.width << a.shift));
  const int64_t pos = length - (end - begin) + (t - begin);
  float q[E], o[E] = {}, m = -INFINITY, d = 0.0f;
  for (int e = 0; e < E; ++e) q[e] = bf2f(a.q[t * a.q_row + head * a.q_head + lane + 64 * e]);
  for (int64_t j = wave; j <= pos; j += 4) {
    const int32_t page = a.table[r * a.table_stride + (j >> a.shift)];
    if (page < 0 || page >= a.pages) continue;
    const int64_t at = page * a.page_stride + (j & ((1 << a.shift) - 1)) * a.row_stride + kvh * a.head_stride + lane;
    float s = 0.0f;
    for (int e = 0; e < E; ++e) s = __builtin_fmaf(q[e], bf2f(a.keys[at + 64 * e]), s);
    for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x, 64);
    s *= a.scale;
    const float mn = fmaxf(m, s), keep = m == mn ? 1.0f : expf(m - mn), p = expf(s - mn);
    d = d * keep + p;
    for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(p, bf2f(a.values[at + 64 * e]), o[e] * keep);
    m = mn;
  }
  if (lane == 0) ms[wave] = m, ds[wave] = d;
  for (int e = 0; e < E; ++e) os[wave][lane + 64 * e] = o[e];
  __syncthreads();
  float M = -INFINITY, D = 0.0f;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, ms[w]);
  for (int c = threadIdx.x; c < HD; c += kSimpleThreads) {
    float x = 0.0f;
    D = 0.0f;
    for (int w = 0; w < 4; ++w) {
      if (ds[w] == 0.0f) continue;
      const float f = expf(ms[w] - M);
      D += ds[w] * f, x += os[w][c] * f;
    }
    x = D == 0.0f ? 0.0f : x / D;
    if (a.gate) x *= 1.0f / (1.0f + expf(-bf2f(a.gate[t * a.gate_row + head * a.gate_head + c])));
    a.out[t * a.out_row + head * a.out_head + c] = f2bf(x);
  }
}

}  // namespace cq35
