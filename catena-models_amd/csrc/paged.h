// Operators of a paged KV cache: pages and slots of a round of requests
// (k_page_plan), and head norm + rotation of a round's projections with the
// keys and values written to their slots (k_paged_prepare).
#pragma once

#include "layers.h"
#include "paged_index.h"

namespace cq35 {

// ------------------------------------------------------------- page plan
//
// With have = ceil(cached / P) and want = ceil(length / P) pages per request,
// the exclusive sums over the requests of max(length - cached, 0),
// max(want - have, 0) and max(have - want, 0) place every new row, page taken
// and page given back. The pages given back lie on the stack above the
// `free` ones in request order; the k-th page taken (request order, then table
// order) is stack[top - 1 - k] with top = free + given back. A new page's
// first row is its request's row at position (page index) * P, so the thread
// of that row writes the table entry and every row finds its page from the
// sums alone.
//
// Nothing a thread reads is written by another: stack entries below `free`
// are read, those from `free` on written; tables are read in columns below
// `have` and written from `have` on; the count in and out are two words. So
// one launch does it, each block repeating the sums over the requests (a few
// KB from L2) instead of waiting for a block that makes them.
//
// Latency-bound: 3.7 us for 8 requests, 7.3 us for 500 with 27 thousand rows,
// 6.1 us for 64 prompts with 99 thousand (an empty launch takes about 2; the
// sums' loads, their two reductions and the rows' search are the rest).
constexpr int kPlanThreads = 256;
constexpr int kPlanMostRequests = 8192;

struct PlanArgs {
  int32_t* table;
  int64_t table_stride;
  int requests;
  int64_t width;
  const int32_t* cached;
  const int32_t* lengths;
  int32_t* stack;
  int64_t pages;
  const int32_t* free_count;
  int shift;
  int64_t rows;
  int32_t* row_start;
  int32_t* positions;
  int32_t* slots;
  int32_t* free_left;
  int32_t* status;
};

inline size_t plan_lds_bytes(int requests) { return ((size_t)requests + 1) * 3 * sizeof(int32_t); }

__global__ __launch_bounds__(kPlanThreads) void k_page_plan(PlanArgs a) {
  extern __shared__ int32_t plan_lds[];
  __shared__ int64_t part[3][kPlanThreads / 64];
  __shared__ int any_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, R = a.requests;
  int32_t *row_s = plan_lds, *take_s = row_s + R + 1, *give_s = take_s + R + 1;
  if (tid == 0) any_bad = 0;
  __syncthreads();
  // each thread a run of requests: its sums, then the exclusive sums of all
  const int per = (R + kPlanThreads - 1) / kPlanThreads;
  const int first = tid * per, last = min(first + per, R);
  int64_t sum[3] = {0, 0, 0};
  bool bad = false;
  for (int r = first; r < last; ++r) {
    const PlanNeed n = plan_need(a.cached[r], a.lengths[r], a.width, a.shift);
    bad |= n.bad;
    sum[0] += n.rows, sum[1] += n.take, sum[2] += n.give;
  }
  if (bad) any_bad = 1;
  int64_t upto[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    int64_t x = sum[i];
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up(x, d, 64);
      if (lane >= d) x += y;
    }
    if (lane == 63) part[i][wave] = x;
    upto[i] = x - sum[i];
  }
  __syncthreads();
  int64_t total[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    total[i] = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      if (w < wave) upto[i] += part[i][w];
      total[i] += part[i][w];
    }
  }
  const int64_t free_pages = *a.free_count;
  const PlanVerdict v = plan_verdict(any_bad != 0, free_pages, a.pages, total[0], total[1], total[2], a.rows);
  const bool ok = v.code == kPlanOk;
  if (ok) {
    for (int r = first; r < last; ++r) {
      const PlanNeed n = plan_need(a.cached[r], a.lengths[r], a.width, a.shift);
      row_s[r] = (int32_t)upto[0], take_s[r] = (int32_t)upto[1], give_s[r] = (int32_t)upto[2];
      upto[0] += n.rows, upto[1] += n.take, upto[2] += n.give;
    }
    if (tid == 0) row_s[R] = (int32_t)total[0], take_s[R] = (int32_t)total[1], give_s[R] = (int32_t)total[2];
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int r = tid; r <= R; r += kPlanThreads) a.row_start[r] = ok ? row_s[r] : 0;
    if (tid == 0) {
      *a.free_left = (int32_t)(ok ? free_pages + total[2] - total[1] : free_pages);
      a.status[0] = v.code;
      a.status[1] = (int32_t)min(v.missing, (int64_t)INT32_MAX);
    }
  }
  const int64_t step = (int64_t)gridDim.x * kPlanThreads, at = (int64_t)blockIdx.x * kPlanThreads + tid;
  const int64_t top = free_pages + total[2];
  // the m-th page given back: the request that loses it, behind what it keeps
  auto given = [&](int64_t m) {
    const int r = request_of(give_s, R, m);
    return a.table[r * a.table_stride + pages_of(a.lengths[r], a.shift) + (m - give_s[r])];
  };
  for (int64_t t = at; t < a.rows; t += step) {
    if (!ok || t >= total[0]) {  // rows behind the last request's
      a.positions[t] = 0;
      a.slots[t] = -1;
      continue;
    }
    const int r = request_of(row_s, R, t);
    const int64_t cached = a.cached[r], pos = cached + (t - row_s[r]);
    const int64_t have = pages_of(cached, a.shift), j = pos >> a.shift;
    int32_t* entry = a.table + r * a.table_stride + j;
    int32_t page;
    if (j < have) {
      page = *entry;
    } else {
      const int64_t i = top - 1 - (take_s[r] + (j - have));
      page = i < free_pages ? a.stack[i] : given(i - free_pages);
      if ((pos & ((1 << a.shift) - 1)) == 0) *entry = page;
    }
    a.positions[t] = (int32_t)pos;
    a.slots[t] = slot_of(page, a.pages, pos, a.shift);
  }
  if (!ok) return;
  const int64_t left = top - total[1];
  for (int64_t m = at; free_pages + m < left && m < total[2]; m += step) a.stack[free_pages + m] = given(m);
}

// ------------------------------------------------- head norm, rotation, append
//
// y = x w / sqrt(mean(x^2) + eps) per query and key head; channels i and
// i + rope_dim / 2 of the first rope_dim are turned by the angle
// position[axis_i] * inv_freq[i]; queries go to q_out, keys and the unchanged
// values to their cache rows. F32 throughout, each result rounded to BF16
// once. The angle is the product taken modulo a turn in 64 bits: an F32 angle is
// off by up to 2^-24 of itself, a sixteenth of a radian at position 10^6. Here
// the product (exact below position 2^29), 1 / (2 pi) and their product are each
// off by at most 2^-53 of the turns, the remainder's rounding to F32 by 2^-26 of
// a turn: together 2^-26 up to 2^20 turns or so, below 2^-22 of a turn at
// position 2^31 - 1 with a frequency of 1.
//
// A head is head_dim / 8 lanes of 16 bytes; a block takes `tokens` rows, makes
// their cosines and sines once in LDS (one pair per thread) and deals the
// rows' heads to its waves, each reading its next head while it works on one.
// HBM-bound: 8192 rows of 16 + 2 + 2 heads of 256 take 40 us, 4.2 TB/s (a large
// copy: 4.9); 2048 blocks of four rows against 1024 of eight: 40 and 55 us.
// Few rows are latency-bound, 7 us for 16 to 777.
constexpr int kPrepThreads = 256;
constexpr int kPrepMostPairs = 128;
constexpr int kPrepMostTokens = 8;
constexpr int kPrepBlocks = 2048;  // eight a CU; more rows share a block's cosines

struct PrepareArgs {
  const uint16_t *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  uint16_t* out;
  int64_t out_row, out_head;
  uint16_t *keys, *values;
  int64_t pages, page_stride, row_stride, head_stride;
  int shift;
  int64_t rows;
  int q_heads, kv_heads, rope_dim;
  const float *q_weight, *k_weight;
  float eps;
  const float* inv_freq;
  const int32_t* positions;
  int64_t position_stride;
  const int32_t* slots;
  int tokens;  // rows of a block
  uint8_t axis[kPrepMostPairs];
};

__device__ __forceinline__ uint32_t pack_bf(float lo, float hi) { return (uint32_t)f2bf(lo) | ((uint32_t)f2bf(hi) << 16); }

template <int HD>
__global__ __launch_bounds__(kPrepThreads) void k_paged_prepare(PrepareArgs a) {
  constexpr int kLanes = HD / 8;                  // lanes of a head
  constexpr int kUnits = kPrepThreads / kLanes;   // heads of a block at a time
  __shared__ float2 turn[kPrepMostTokens][kPrepMostPairs];
  const int tid = threadIdx.x, c = tid % kLanes, half = a.rope_dim / 2;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n = (int)min((int64_t)a.tokens, a.rows - t0);
  const int heads = a.q_heads + 2 * a.kv_heads;
  // a head of a row: read ahead of the one being worked on
  struct Unit {
    int t, h;
    int32_t slot;
    u32x4 raw;
  };
  auto read = [&](Unit& u) {
    const int64_t row = t0 + u.t;
    u.slot = a.slots[row];
    const int g = u.h - a.q_heads;
    const uint16_t* src = g < 0 ? a.q + row * a.q_row + u.h * a.q_head
                          : g < a.kv_heads ? a.k + row * a.k_row + g * a.k_head
                                           : a.v + row * a.v_row + (g - a.kv_heads) * a.v_head;
    u.raw = *reinterpret_cast<const u32x4*>(src + 8 * c);
  };
  auto advance = [&](Unit& u) {
    for (u.h += kUnits; u.h >= heads; u.h -= heads) ++u.t;
  };
  Unit next = {0, tid / kLanes, -1, {}};
  for (; next.h >= heads; next.h -= heads) ++next.t;
  if (next.t < n) read(next);
  float wq[8], wk[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 x = reinterpret_cast<const float4*>(a.q_weight + 8 * c)[i], y = reinterpret_cast<const float4*>(a.k_weight + 8 * c)[i];
    wq[4 * i] = x.x, wq[4 * i + 1] = x.y, wq[4 * i + 2] = x.z, wq[4 * i + 3] = x.w;
    wk[4 * i] = y.x, wk[4 * i + 1] = y.y, wk[4 * i + 2] = y.z, wk[4 * i + 3] = y.w;
  }
  for (int i = tid; i < n * half; i += kPrepThreads) {
    const int t = i / half, p = i - t * half;
    const double product = (double)a.positions[a.axis[p] * a.position_stride + t0 + t] * (double)a.inv_freq[p];
    double turns = product * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, co;
    sincospif(2.0f * (float)turns, &s, &co);
    turn[t][p] = make_float2(co, s);
  }
  __syncthreads();
  while (next.t < n) {
    const Unit u = next;
    advance(next);
    if (next.t < n) read(next);
    if (u.slot < 0 || (u.slot >> a.shift) >= a.pages) continue;  // the same for every lane of the head
    const int64_t cache_row = (int64_t)(u.slot >> a.shift) * a.page_stride + (int64_t)(u.slot & ((1 << a.shift) - 1)) * a.row_stride + 8 * c;
    const int g = u.h - a.q_heads;
    if (g >= a.kv_heads) {
      *reinterpret_cast<u32x4*>(a.values + cache_row + (g - a.kv_heads) * a.head_stride) = u.raw;
      continue;
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = lo2f(u.raw[i]), x[2 * i + 1] = hi2f(u.raw[i]);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(x[i], x[i], sum);
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) sum += __shfl_xor(sum, d, 64);
    const float inverse = 1.0f / sqrtf(sum * (1.0f / HD) + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * inverse * (g < 0 ? wq[i] : wk[i]);
    // the pairs' other channels lie rope_dim / 16 lanes away
    const int away = half / 8, lane = tid & 63;
    const bool front = c < away, turned = c < 2 * away;
    const int from = turned ? (front ? lane + away : lane - away) : lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = __shfl(x[i], from, 64);
      if (turned) {
        const float2 r = turn[u.t][8 * (front ? c : c - away) + i];
        x[i] = front ? x[i] * r.x - o * r.y : x[i] * r.x + o * r.y;
      }
    }
    u32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = pack_bf(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<u32x4*>(g < 0 ? a.out + (t0 + u.t) * a.out_row + u.h * a.out_head + 8 * c : a.keys + cache_row + g * a.head_stride) = y;
  }
}

}  // namespace cq35
