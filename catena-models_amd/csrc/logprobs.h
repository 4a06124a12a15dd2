// Log probabilities of given tokens, entropy and the most likely tokens of rows of
// logits, in one pass over them.
#pragma once

#include "lanes.h"
#include "layers.h"

namespace cq35 {

// With m = max x, s = sum e^(x - m) and t = sum e^(x - m) (x - m) of a row:
//   log p_i = (x_i - m) - log s,   entropy = log s - t / s.
// (m, s, t) of two parts of a row join to M = max(m, m'), s f + s' f' and
// f (t + s (m - M)) + f' (t' + s' (m' - M)) with f = e^(m - M), so a row can be cut
// anywhere: k_logprobs runs a block over a run of a row's tiles and, where a row
// has several blocks, leaves (m, s, t) and the block's best tokens for
// k_logprobs_join.
//
// The best tokens: every logit has a key of 64 bits, its order as a number and, among
// equal ones, its place, so no two are equal and the order in which candidates
// are found changes nothing. A block keeps candidates in LDS and a threshold, the
// top-th best key so far, for the next kEpoch tiles; a thread looks at its logits of a
// tile one by one only if the largest passes it. Without a threshold yet one is taken
// from the threads' largest logits (group_bound). Where more candidates pass than the
// list holds (rows that ascend), the tiles are looked at again one by
// one, where many threads have any over the top-th of the 256 threads' largest keys: at most 32 logits of each of
// top threads reach it. So is a tile alone whose bound many groups' largest logits equal (a mask's
// lowest value, rows of equal logits): its keys' threshold serves the rest.
// 64 rows of F32 with 20, 99.9 of 100 logits masked, 34 us in all instead of 23, and 90 with each
// such tile's equal logits as candidates; whole keys instead of orders in group_bound 28, but then 27.5 for rows
// without a mask.
//
// Bound by the logits' bytes where there are many rows: 1000 rows of 248320 BF16 logits with one
// alternative 95 us (5.2 TB/s), with 20 105; 64 rows of F32 with 20 18.8, without any 12.2. One row is
// latency: 6.8 us in 31 blocks, then 4 us for the join. A row is cut into as many blocks as 1024 hold of all rows, so
// beyond 512 rows each has one: 512 rows with 5 take 60 us, 600 take 74; a row beyond 1024 waits for a block that
// ends: 1025 rows with one 111. A barrier a tile: 205 us for the 1000 rows, one in two 8 % and one in four 2 % more
// than one in eight, one in sixteen as much as in eight. A candidate's logit read again where it is found, and not
// all of them at once in front of best_keys: 102 us; a thread's logits kept in registers for them: 168 registers
// instead of 127, half the waves; tiles of 32 F32 logits a thread instead of 16: spilled, 31 us for the 64 rows; 512
// or 2048 blocks wanted instead of 1024: 75 and 56 us for 300 rows, 53.
constexpr int kLogprobsMostTop = 32;
constexpr int kLogprobsMostGiven = 1024;
constexpr int kLogprobThreads = 256;
constexpr int kLogprobPieces = 4;                                 // of 16 bytes, a thread's share of a tile
constexpr int kCandidates = 2048;                                 // of the list
constexpr int kLogprobMostSplits = kCandidates / kLogprobsMostTop;  // of a row, so that the join's list holds them
constexpr int kEpoch = 8;                                         // tiles between two looks at the list
constexpr int kMoreGroups = 8;                                    // that may pass a bound beside those needed
constexpr int kLogprobPrune = 128;                                // candidates that are cut down to the best
constexpr int kRankedAtOnce = 128;                                // candidates that are ranked without a bound

struct LogprobArgs {
  const void* logits;
  int64_t stride, rows;
  int vocab;
  const int64_t* tokens;
  int given, top;
  float *logprobs, *entropy;
  int64_t* top_tokens;
  float* top_logprobs;
  int splits;          // blocks of a row
  float* stats;        // [rows][splits][4]: m, s, t
  uint64_t* keys;      // [rows][splits][top], 0 behind the last
};

__device__ __forceinline__ float widened(uint16_t x) { return bf2f(x); }
__device__ __forceinline__ float widened(float x) { return x; }

// Larger for larger logits (NaN above infinity, -0 as 0), among equal ones for lower indices;
// never 0.
__device__ __forceinline__ uint32_t order_of_logit(float x) {
  const uint32_t b = fbits(x + 0.0f);
  return x != x ? 0xffffffffu : b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t logit_key(float x, int index) {
  return (uint64_t)order_of_logit(x) << 32 | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ int key_index(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t order = (uint32_t)(key >> 32);
  return bitsf(order >> 31 ? order ^ 0x80000000u : ~order);
}

// s and t of the logits so far, over their maximum m. Exponents are made from x - m: those of one fused
// multiply-add, c x - c m, would save an operation of ten per logit, but c m rounds, and a row of one
// likely token would not have the entropy 0. NaN in s goes on into every result: a row that holds NaN or
// +inf.
struct RowStats {
  float m, s, t;  // m: -inf before any logit
  __device__ __forceinline__ void clear() { m = -__builtin_inff(), s = t = 0.0f; }
  static __device__ __forceinline__ float reference(float m) { return m == -__builtin_inff() ? 0.0f : m; }
  static __device__ __forceinline__ float power(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504f); }
  __device__ __forceinline__ void rebase(float to) {
    const float d = m - reference(to), f = power(d);
    t = f * (t + s * fmaxf(d, -200.0f));
    s *= f, m = to;
  }
  // a logit's terms, d = x - m
  static __device__ __forceinline__ void add(float d, float& s, float& t) {
    const float w = power(d);
    s += w, t = __builtin_fmaf(w, fmaxf(d, -200.0f), t);  // nothing of a logit of -inf
  }
  // of all lanes
  __device__ __forceinline__ void over_wave() {
    rebase(lanes_max(m));
    s = lanes_sum(s), t = lanes_sum(t);
  }
};

struct LogprobShared {
  alignas(16) uint64_t list[kCandidates];
  alignas(16) uint64_t per_thread[kLogprobThreads];
  RowStats stats[kLogprobThreads / 64];
  alignas(16) uint32_t groups[64];
  uint64_t best[kLogprobsMostTop];
  uint64_t exact;
  int count[3], kept;
};

// The top-th largest of the maxima of 64 groups of four threads: as many of the threads' values are not
// below it, and few more. (The least maximum of 4 to 32 larger groups needs no ranks, but five times as many
// pass it.) Ends behind a barrier and reads what lies in front of the next. passed: the groups of the first
// `groups` that are not below it, more than top where many are equal.
__device__ __forceinline__ uint32_t group_bound(LogprobShared& l, uint32_t x, int top, int groups, int& passed) {
  const int lane = threadIdx.x & 63;
  x = max(x, lane_moved<0xb1>(x));
  x = max(x, lane_moved<0x4e>(x));
  if ((lane & 3) == 0) l.groups[threadIdx.x >> 2] = x;
  __syncthreads();
  const uint32_t mine = l.groups[lane];
  int rank = 0;
#pragma unroll
  for (int j = 0; j < 64; j += 4) {
    const uint4 y = *reinterpret_cast<const uint4*>(l.groups + j);
    rank += (y.x > mine) + (y.y > mine) + (y.z > mine) + (y.w > mine);
  }
  passed = __popcll(__ballot(rank < top && lane < groups));
  return over_lanes(rank < top ? mine : 0xffffffffu, [](uint32_t a, uint32_t b) { return min(a, b); });
}

// Every key of that order or a larger one is above the result.
__device__ __forceinline__ uint64_t below_order(uint32_t order) { return order ? ((uint64_t)order << 32) - 1 : 0; }
// A number that logits of that order or a larger one are not at or below, other numbers are: the next one
// down (no logit has the order of -0).
__device__ __forceinline__ float below_logit(uint32_t order) {
  return key_logit((uint64_t)(order == 0x80000000u ? order - 2 : order - 1) << 32);
}

constexpr int kShare = kCandidates / kLogprobThreads;  // of the list, per thread

// How many of the first n keys at `list` are larger than each of the thread's.
template <int kCount>
__device__ __forceinline__ void ranks(const uint64_t* list, int n, const uint64_t (&mine)[kShare], int (&rank)[kShare]) {
#pragma unroll
  for (int b = 0; b < kCount; ++b) rank[b] = 0;
  int j = 0;
#pragma unroll 2
  for (; j + 4 <= n; j += 4) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(list + j), y = *reinterpret_cast<const ulonglong2*>(list + j + 2);
#pragma unroll
    for (int b = 0; b < kCount; ++b) rank[b] += (x.x > mine[b]) + (x.y > mine[b]) + (y.x > mine[b]) + (y.y > mine[b]);
  }
  for (; j < n; ++j)
#pragma unroll
    for (int b = 0; b < kCount; ++b) rank[b] += list[j] > mine[b];
}

// The best min(n, top) of the list's n keys into `best`, in descending order, and into the list's front;
// the threshold that follows, 0 where there are fewer than top. Every thread has to be behind a
// barrier that the list was written in front of; ends behind another.
__device__ __forceinline__ uint64_t best_keys(LogprobShared& l, int n, int top) {
  const int tid = threadIdx.x;
  uint64_t mine[kShare];
  int rank[kShare];
#pragma unroll
  for (int b = 0; b < kShare; ++b) mine[b] = b * kLogprobThreads + tid < n ? l.list[b * kLogprobThreads + tid] : 0;
  if (n > kRankedAtOnce) {  // most are below a bound that is sooner had than their ranks (with 64, 0.5 us more for 64 rows with 20)
    uint32_t most = 0;
#pragma unroll
    for (int b = 0; b < kShare; ++b) most = max(most, (uint32_t)(mine[b] >> 32));
    if (tid == 0) l.kept = 0;
    int passed;
    const uint64_t above = below_order(group_bound(l, most, top, 64, passed));  // a barrier: the list has been read
#pragma unroll
    for (int b = 0; b < kShare; ++b)
      if (mine[b] > above) l.list[atomicAdd(&l.kept, 1)] = mine[b];
    __syncthreads();
    n = l.kept;
#pragma unroll
    for (int b = 0; b < kShare; ++b) mine[b] = b * kLogprobThreads + tid < n ? l.list[b * kLogprobThreads + tid] : 0;
  }
  if (n > kLogprobThreads) ranks<kShare>(l.list, n, mine, rank);
  else if ((tid & ~63) < n) ranks<1>(l.list, n, mine, rank);
#pragma unroll
  for (int b = 0; b < kShare; ++b)
    if (b * kLogprobThreads + tid < n && rank[b] < top) l.best[rank[b]] = mine[b];
  __syncthreads();
  if (tid < min(n, top)) l.list[tid] = l.best[tid];
  return n >= top ? l.best[top - 1] : 0;
}

// What a row's results need beside its statistics, asked for ahead of them.
template <typename T>
struct GivenToken {
  float x;  // the thread's first given token's logit, NaN for no token of the row
  static __device__ __forceinline__ float logit(const LogprobArgs& a, int64_t row, int i) {
    const int64_t token = a.tokens[row * a.given + i];
    return token >= 0 && token < a.vocab ? widened(((const T*)a.logits)[row * a.stride + token]) : __builtin_nanf("");
  }
  __device__ __forceinline__ void load(const LogprobArgs& a, int64_t row) {
    if ((int)threadIdx.x < a.given) x = logit(a, row, threadIdx.x);
  }
  // best: the row's best keys
  __device__ __forceinline__ void finish(const LogprobArgs& a, int64_t row, const RowStats& r, const uint64_t* best) const {
    const float log_s = logf(r.s);
    const int tid = threadIdx.x;
    if (tid == 0) a.entropy[row] = log_s - r.t / r.s;
    for (int i = tid; i < a.given; i += kLogprobThreads)
      a.logprobs[row * a.given + i] = ((i == tid ? x : logit(a, row, i)) - r.m) - log_s;
    if (tid < a.top) {
      const uint64_t key = best[tid];
      a.top_tokens[row * a.top + tid] = key_index(key);
      a.top_logprobs[row * a.top + tid] = (key_logit(key) - r.m) - log_s;
    }
  }
};

// A thread's logits of a tile: pieces of 16 bytes, 256 pieces apart, from the 16-byte address at or
// below the row's start.
template <typename T>
struct LogitTile {
  static constexpr int E = 16 / sizeof(T), kPieces = kLogprobPieces, kLogits = E * kPieces * kLogprobThreads;
  u32x4 raw[kPieces];
  static __device__ __forceinline__ int first(int tile, int j) { return ((tile * kPieces + j) * kLogprobThreads + (int)threadIdx.x) * E; }
  // the same for the whole block
  static __device__ __forceinline__ bool whole(int before, int end, int tile) {
    return tile * kLogits >= before && (tile + 1) * kLogits <= end;
  }
  // -inf in the places outside the row
  static __device__ __forceinline__ u32x4 edge(const T* base, int before, int end, int i) {
    if (i >= before && i + E <= end) return *reinterpret_cast<const u32x4*>(base + i);
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = i + e >= before && i + e < end ? widened(base[i + e]) : -__builtin_inff();
    u32x4 x;
#pragma unroll
    for (int w = 0; w < 4; ++w) x[w] = E == 8 ? fbits(v[2 * w % E]) >> 16 | (fbits(v[(2 * w + 1) % E]) & 0xffff0000u) : fbits(v[w % E]);
    return x;
  }
  __device__ __forceinline__ void load(const T* base, int before, int end, int tile) {
    if (whole(before, end, tile)) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) raw[j] = *reinterpret_cast<const u32x4*>(base + first(tile, j));
    } else {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) raw[j] = edge(base, before, end, first(tile, j));
    }
  }
  // f(logit, index) of each of the share, read again: unrolled for the few tiles that need it, what is
  // done with them would halve the waves
  template <typename F>
  static __device__ __forceinline__ void each(const T* base, int before, int end, int tile, F f) {
#pragma unroll 1
    for (int j = 0; j < kPieces; ++j) {
      LogitTile one;
      const int i = first(tile, j);
      one.raw[0] = edge(base, before, end, i);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e >= before && i + e < end) f(one.value(0, e), i + e - before);
    }
  }
  __device__ __forceinline__ float value(int j, int e) const {
    return E == 4 ? bitsf(raw[j][e & 3]) : e & 1 ? hi2f(raw[j][e >> 1]) : lo2f(raw[j][e >> 1]);
  }
};

template <typename T, bool kTop>
__global__ __launch_bounds__(kLogprobThreads, 4) void k_logprobs(LogprobArgs a) {
  typedef LogitTile<T> Tile;
  __shared__ LogprobShared l;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / (uint32_t)a.splits;
  const int split = blockIdx.x % (uint32_t)a.splits;
  const T* x = (const T*)a.logits + row * a.stride;
  // places counted from the aligned address: the row is before .. end
  const int before = (int)(((uintptr_t)x & 15) / sizeof(T)), end = before + a.vocab;
  const T* base = x - before;
  const int tiles = (end + Tile::kLogits - 1) / Tile::kLogits;
  const int t0 = (int)((int64_t)tiles * split / a.splits), t1 = (int)((int64_t)tiles * (split + 1) / a.splits);
  if (tid < 3) l.count[tid] = 0;
  __syncthreads();
  GivenToken<T> given;
  if (a.splits == 1) given.load(a, row);
  RowStats r;
  r.clear();
  uint64_t threshold = 0;         // the top-th best key so far
  float limit = 0.0f;             // logits not at or below it are candidates
  int n = 0, keys = 0, turn = 0;  // in the list; of them keys, the others still places; which count is in use
  auto put = [&](uint64_t key) {
    const int at = n + atomicAdd(&l.count[turn], 1);
    if (at < kCandidates) l.list[at] = key;
  };
  auto added = [&] {
    const int next_turn = turn == 2 ? 0 : turn + 1;
    if (tid == 0) l.count[next_turn] = 0;  // last read two barriers ago
    __syncthreads();
    const int c = l.count[turn];
    turn = next_turn;
    return c;
  };
  Tile next;
  if (t0 < t1) next.load(base, before, end, t0);
  for (int tile = t0; tile < t1;) {
    const int start = tile;
    int stop = min(tile + kEpoch, t1);
#pragma unroll 1
    for (; tile < stop; ++tile) {
      const Tile v = next;
      if (tile + 1 < t1) next.load(base, before, end, tile + 1);
      float most = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < Tile::kPieces; ++j)
#pragma unroll
        for (int e = 0; e < Tile::E; ++e) most = fmaxf(most, v.value(j, e));
      if (most > r.m) r.rebase(most);
      // a tile's terms first among themselves: one chain over a row's logits rounds a thousand times, and
      // loses terms below half a step of the sum
      const float from = RowStats::reference(r.m);
      float tile_s = 0.0f, tile_t = 0.0f;
#pragma unroll
      for (int j = 0; j < Tile::kPieces; ++j)
#pragma unroll
        for (int e = 0; e < Tile::E; ++e) RowStats::add(v.value(j, e) - from, tile_s, tile_t);
      r.s += tile_s, r.t += tile_t;
      if (!kTop) continue;
      if (threshold == 0 && tile == start) {
        int passed;
        const uint32_t order = group_bound(l, order_of_logit(most), a.top, (end - tile * Tile::kLogits + 4 * Tile::E - 1) / (4 * Tile::E), passed);
        limit = below_logit(order);
        // of equal logits far more would pass than are wanted: none is taken, and the tile is looked at again at once
        if (passed > a.top + kMoreGroups) limit = __builtin_inff(), stop = tile + 1;
      }
      if (!(most <= limit) || r.s != r.s) {
        // which of the logits pass: their places, as few do and a wait for one read again would be the tile's
        uint32_t pass = 0;
#pragma unroll
        for (int j = Tile::kPieces - 1; j >= 0; --j) {
          // a piece at a time and only here: all of it made ahead takes 80 registers more
          LogitTile<T> one;
          one.raw[0] = v.raw[j];
          asm volatile("" : "+v"(one.raw[0]), "+v"(pass));
#pragma unroll
          for (int e = Tile::E - 1; e >= 0; --e) pass = 2 * pass + (one.value(0, e) <= limit ? 0 : 1);
        }
        for (; pass; pass &= pass - 1) {
          const int at = __builtin_ctz(pass), i = Tile::first(tile, at / Tile::E) + at % Tile::E;
          if (i >= before && i < end) put(i);
        }
      }
    }
    if (!kTop) continue;
    if (tid == 0 && limit == __builtin_inff()) l.count[turn] = kCandidates + 1;
    const int c = added();
    const bool many = n + c > kCandidates;
    if (!many) n += c;
    if (many || tile == t1 || n >= kLogprobPrune || (threshold == 0 && n >= a.top)) {
      // all of the places' logits at once
      for (int i = tid; i < n; i += kLogprobThreads)
        if (i >= keys) l.list[i] = logit_key(widened(base[l.list[i]]), (int)l.list[i] - before);
      __syncthreads();
      if (!many) {
        threshold = best_keys(l, n, a.top);
        n = min(n, a.top);
      } else {
#pragma unroll 1
        for (int again = start; again < stop; ++again) {
          uint64_t own = 0;
          Tile::each(base, before, end, again, [&](float x, int i) { own = max(own, logit_key(x, i)); });
          l.per_thread[tid] = own;
          if (tid == 0) l.exact = 0;
          const int over = __syncthreads_count(own > threshold);
          if (over == 0) continue;
          uint64_t above = threshold;
          if (n + over * Tile::kPieces * Tile::E > kCandidates) {  // the list might not hold what these threads have
            // the top-th of the threads' largest keys
            uint64_t mine[kShare];
            int rank[kShare];
            mine[0] = own;
            ranks<1>(l.per_thread, kLogprobThreads, mine, rank);
            if (own && rank[0] == a.top - 1) l.exact = own - 1;
            __syncthreads();
            above = max(l.exact, threshold);
          }
          Tile::each(base, before, end, again, [&](float x, int i) {
            const uint64_t key = logit_key(x, i);
            if (key > above) put(key);
          });
          n += added();
          threshold = best_keys(l, n, a.top);
          n = min(n, a.top);
        }
      }
      keys = n;
    }
    if (threshold) limit = key_logit(threshold);
  }
  r.over_wave();
  if ((tid & 63) == 0) l.stats[tid >> 6] = r;
  __syncthreads();
  r = l.stats[tid & 3];
  r.over_wave(), r.s *= 1.0f / 16, r.t *= 1.0f / 16;  // each wave's in 16 lanes
  if (a.splits == 1) {
    given.finish(a, row, r, l.best);
    return;
  }
  if (tid == 0) *reinterpret_cast<float4*>(a.stats + 4 * (int64_t)blockIdx.x) = make_float4(r.m, r.s, r.t, 0.0f);
  if (kTop && tid < a.top) a.keys[(int64_t)blockIdx.x * a.top + tid] = tid < n ? l.best[tid] : 0;
}

// A block a row: its parts' statistics in the lanes of a wave, their best keys in the threads.
template <typename T>
__global__ __launch_bounds__(kLogprobThreads) void k_logprobs_join(LogprobArgs a) {
  __shared__ LogprobShared l;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int n = a.splits * a.top;
  // the parts' best keys go to threads of different groups; 0 behind the last
  const int filled = (n + kLogprobThreads - 1) / kLogprobThreads * kLogprobThreads;
#pragma unroll
  for (int b = 0; b < kShare; ++b) {
    const int at = b * kLogprobThreads + tid, i = b * kLogprobThreads + (tid & 3) * 64 + (tid >> 2);
    if (at < filled) l.list[at] = i < n ? a.keys[row * n + i % a.splits * a.top + i / a.splits] : 0;
  }
  GivenToken<T> given;
  given.load(a, row);
  RowStats r;
  r.clear();
  if ((tid & 63) < a.splits) {
    const float4 p = *reinterpret_cast<const float4*>(a.stats + 4 * (row * a.splits + (tid & 63)));
    r = {p.x, p.y, p.z};
  }
  r.over_wave();
  if (a.top) {
    __syncthreads();
    best_keys(l, filled, a.top);
  }
  given.finish(a, row, r, l.best);
}

}  // namespace cq35
