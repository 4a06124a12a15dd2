// Attention of new tokens over a paged KV cache, on the matrix cores: scores
// S^T = K Q^T of 32 keys and 32 packed rows (row * group + query head), the
// running maximum and sum of a softmax per row, O^T += V^T P^T.
//
// v_mfma_f32_32x32x16_bf16 (operand layouts: mfma.h) leaves the 16 scores of a
// lane all in one row's column, so that maxima and sums are in-lane but for
// one exchange of the two half-waves, and the weights, rounded to BF16, lie
// where the second product takes them: register 8 s + i of half h is key
// 16 s + 8 (i / 4) + 4 h + i % 4. V^T's operand for those keys is two
// ds_read_b64_tr_b16, each of which hands lane j of 16 the 4 keys x 1 channel
// that lanes 4 e .. 4 e + 3 point at as 4 channels of key e.
//
// Key and value tiles go straight to LDS (16 bytes a lane, no registers held)
// in rows of head_dim, their 16-byte pieces swizzled by the row so that the 32
// rows of a key operand and the 8 rows of a value operand spread over the
// banks.
//
// The weights' rounding to BF16 (at most 2^-8 of each, as the values' own) takes
// a sixteenth of the time that products of F32 weights would;
// the sum of the weights takes them unrounded, in F32. A row's maximum moves
// only when it grows by more than 8 (in units of a factor 2; the first tile
// aside): weights stay below 2^8, exact to scale in BF16 and F32, and the
// sums are not rescaled at every tile.
//
// Zero weights do not hide a non-finite value of a later token from the rows
// in front of it (0 * inf). A row whose result is NaN is therefore done again
// with the keys behind its position left out of the tiles: only calls with
// such values, or with NaN results, pay for it. Rows behind a request's end
// and those of pages outside the cache are never read: zeros take their place.
#pragma once

#include <algorithm>
#include <type_traits>

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
  int64_t table_stride;
  const int32_t *row_start, *lengths;
  int requests;
  // |scale| log2(e): scores in units of a factor 2. The scale's sign goes into
  // the queries' (a scale of 0: queries of 0, scaled by 1), so that masked
  // scores of -inf stay that.
  float scale2;
  uint32_t q_and, q_xor;
  CutRule cut;
  float* part;   // slots of [group of 32 rows]: weighted sums in fragment order, then maxima, then sums
};

constexpr float kRescale = 8.0f;

// ------------------------------------------------------------ finding work

struct Found {
  int32_t request, index;  // the request and the item (or row tile) inside it
  int64_t parts_before;    // partial results of earlier requests
  int32_t chunk;
};

// Inclusive sums over the lanes of a wave (rows of 16 by shifts, then the rows'
// ends handed on); every lane active.
template <int kCtrl, int kRows>
__device__ __forceinline__ int64_t lanes_moved(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, kCtrl, kRows, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)((uint64_t)x >> 32), kCtrl, kRows, 0xf, false);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t wave_sums(int64_t x) {
  x += lanes_moved<0x111, 0xf>(x);  // row_shr:1
  x += lanes_moved<0x112, 0xf>(x);
  x += lanes_moved<0x114, 0xf>(x);
  x += lanes_moved<0x118, 0xf>(x);
  x += lanes_moved<0x142, 0xa>(x);  // row_bcast:15 into rows 1 and 3
  x += lanes_moved<0x143, 0xc>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)x >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// The request that holds item `at` (kTiles: row tile `at`) of the launch, in
// uniform registers. Every block makes the sums over all requests itself, 64
// of them in the lanes of a wave: up to 64 requests without a barrier (a
// decode item of 16 keys would otherwise wait for three), and no launch in
// front of this one.
constexpr int kAttendMostRequests = 8192;
template <bool kTiles, int kThreads>
__device__ __forceinline__ bool find_work(const AttendArgs& a, uint32_t at, Found* found, CutRequest* req) {
  constexpr int W = kThreads / 64, kSlices = kAttendMostRequests / 64;
  __shared__ int64_t sums[3][kSlices];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, R = a.requests, slices = (R + 63) / 64;
  auto shape = [&](int slice) {
    const int r = 64 * slice + lane;
    CutRequest q = {};
    if (r < R) q = cut_request(a.cut, a.row_start[r], a.row_start[r + 1], a.lengths[r]);
    return q;
  };
  auto work_of = [&](const CutRequest& q) { return request_work(a.cut, q); };
  auto items_of = [&](const CutRequest& q, int n) { return kTiles ? q.tiles : (int64_t)q.tiles * n; };
  auto parts_of = [](const CutRequest& q, int n) { return n > 1 ? (int64_t)q.tiles * n : 0; };
  CutRequest q;
  int slice = 0, chunk;
  int64_t before = 0, parts_before = 0;  // of earlier slices
  if (slices == 1) {
    q = shape(0);
    chunk = cut_chunk(a.cut, lane_value(wave_sums(work_of(q)), 63), [&](int32_t x) {
      return lane_value(wave_sums((int64_t)q.tiles * cut_splits(a.cut, q, x)), 63);
    });
  } else {
    for (int s = wave; s < slices; s += W) {
      const int64_t x = wave_sums(work_of(shape(s)));
      if (lane == 63) sums[0][s] = x;
    }
    __syncthreads();
    int64_t pairs = 0;
    for (int s = lane; s < slices; s += 64) pairs += sums[0][s];
    CutRule plain = a.cut;
    plain.search = 0;
    chunk = cut_chunk(plain, lane_value(wave_sums(pairs), 63), [](int32_t) { return (int64_t)0; });
    for (int s = wave; s < slices; s += W) {
      q = shape(s);
      const int n = cut_splits(a.cut, q, chunk);
      const int64_t x = wave_sums(items_of(q, n)), y = wave_sums(parts_of(q, n));
      if (lane == 63) sums[1][s] = x, sums[2][s] = y;
    }
    __syncthreads();
    for (;; slice += 64) {  // 64 slices at a time
      if (slice >= slices) return false;
      const bool in = slice + lane < slices;
      const int64_t own = in ? sums[1][slice + lane] : 0, parts = in ? sums[2][slice + lane] : 0;
      const int64_t upto = wave_sums(own), parts_upto = wave_sums(parts);
      const uint64_t past = __ballot(at < before + upto);
      const int hit = past ? __builtin_ctzll(past) : 63;
      if (past) {
        before += lane_value(upto - own, hit), parts_before += lane_value(parts_upto - parts, hit);
        slice += hit;
        break;
      }
      before += lane_value(upto, 63), parts_before += lane_value(parts_upto, 63);
    }
    q = shape(slice);
  }
  const int n = cut_splits(a.cut, q, chunk);
  const int64_t own = items_of(q, n), parts = parts_of(q, n), upto = wave_sums(own), parts_upto = wave_sums(parts);
  const uint64_t past = __ballot(at < before + upto);
  if (!past) return false;
  const int hit = __builtin_ctzll(past);
  found->request = 64 * slice + hit;
  found->index = (int32_t)(at - before - lane_value(upto - own, hit));
  found->parts_before = parts_before + lane_value(parts_upto - parts, hit);
  found->chunk = chunk;
  auto value = [&](int32_t x) { return __builtin_amdgcn_readlane(x, hit); };
  *req = {value(q.begin), value(q.end), lane_value(q.lead, hit), value(q.length), value(q.packed), value(q.tiles), value(q.key_tiles)};
  return true;
}

// ------------------------------------------------------------ tiles in LDS

template <int HD>
struct KvTile {
  static constexpr int kRow = 2 * HD;               // bytes of a row
  static constexpr int kBytes = kKeyTile * kRow;    // of a tile of keys, or of values
  static constexpr int kPieces = HD / 8;            // 16-byte pieces of a row
  static constexpr int kLoads = kBytes / 1024;      // wave-wide requests of a tile
  static constexpr int kPer = 1024 / kRow;          // rows of a request
  static __device__ __forceinline__ int key_swizzle(int row) { return row & (kPieces < 16 ? kPieces - 1 : 15); }
  static __device__ __forceinline__ int value_swizzle(int row) {
    return HD == 64 ? (row >> 1 & 1) << 2 : (row & (kPieces / 4 - 1)) << 2;
  }
};

// The lane's number, made anew: what follows from it is not kept in registers
// around a loop that has none to spare.
__device__ __forceinline__ int lane_here() {
  int l = threadIdx.x & 63;
  asm volatile("" : "+v"(l));
  return l;
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// 16 bytes per lane from `from` to LDS `to` + 16 lane. Written out because the
// compiler would make every later LDS read wait for all of them.
__device__ __forceinline__ void request_lds(uint32_t to, const void* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}

// The same from a uniform base and a lane's offset in bytes.
__device__ __forceinline__ void request_lds(uint32_t to, const void* base, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(to), "v"(offset), "s"(base)
               : "memory", "m0");
}

// All but the newest `n` requests of this wave have arrived.
template <int n>
__device__ __forceinline__ void arrived_but() {
  static_assert(n >= 0 && n < 64, "the counter's range");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0f70 | (n & 15) | ((n >> 4) << 14));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Where keys lie: runs of 16 rows, each in one page (pages hold a multiple of
// 16). A window keeps the places of the runs of 32 tiles, `step` tiles apart, in
// the lanes of a wave (lane 2 i + h: run h of the window's tile i), as bytes
// from the cache's base: a table entry read for every tile would be waited for
// with the tile's LDS reads, which share its counter, and its products cost as
// many scalar instructions as a tile's softmax has vector ones. Runs of pages
// outside the cache and of tiles from `end` on are bad and lie nowhere.
struct Window {
  uint32_t lo, hi;
  uint64_t bad;
  // tiles first, first + step, ...
  __device__ __forceinline__ void fill(const AttendArgs& a, int request, int64_t kv_offset, int first, int step, int end,
                                       int last_key) {
    const int lane = lane_here(), tile = first + (lane >> 1) * step;
    // the second run of the last tile may lie behind the last key, where the
    // table may end; its rows are not read
    const int key = min(kKeyTile * min(tile, end - 1) + 16 * (lane & 1), last_key);
    const int32_t page = a.table[request * a.table_stride + (key >> a.shift)];
    const bool none = tile >= end || page < 0 || page >= a.pages;
    const int row = (key & ~15) & ((1 << a.shift) - 1);
    const int64_t at = none ? 0 : 2 * (page * a.page_stride + row * a.row_stride + kv_offset);
    lo = (uint32_t)at, hi = (uint32_t)((uint64_t)at >> 32);
    bad = __ballot(none);
  }
  __device__ __forceinline__ int64_t at(int run) const {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, run) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, run));
  }
};

// Zeros in place of rows that must not be read.
__device__ __align__(16) uint32_t attend_zeros[4];

// `count` requests of the rows from `row` (of the tile) of a run at byte `at`,
// into the tile at LDS `to`; zeros for rows behind `last_row` of the tile, and
// for a bad run.
template <int HD, bool kKeys>
__device__ __forceinline__ void request_rows(const AttendArgs& a, int64_t at, bool bad, int row0, int last_row, uint32_t to,
                                             int count) {
  typedef KvTile<HD> T;
  const int lane = lane_here(), lr = lane / T::kPieces, piece = lane % T::kPieces;
  const uint8_t* base = reinterpret_cast<const uint8_t*>(kKeys ? a.keys : a.values) + at;
  const int rs = 2 * (int)a.row_stride;
  to += row0 * T::kRow;
  if (!bad && last_row >= row0 + count * T::kPer - 1) {
    base += (int64_t)(row0 & 15) * rs;
#pragma unroll
    for (int n = 0; n < count; ++n) {
      const int row = row0 + n * T::kPer + lr;
      request_lds(to + 1024 * n, base, lr * rs + 16 * (piece ^ (kKeys ? T::key_swizzle(row) : T::value_swizzle(row))));
      base += (int64_t)T::kPer * rs;
    }
  } else {
#pragma unroll 1
    for (int n = 0; n < count; ++n) {
      const int row = row0 + n * T::kPer + lr;
      const int off = 16 * (piece ^ (kKeys ? T::key_swizzle(row) : T::value_swizzle(row)));
      const uint8_t* from = base + (int64_t)(row & 15) * rs + off;
      request_lds(to + 1024 * n, bad || row > last_row ? reinterpret_cast<const uint8_t*>(attend_zeros) : from);
    }
  }
}

// ------------------------------------------------------------ one tile

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The other half-wave's value of the same column.
__device__ __forceinline__ float other_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_weights(float a, float b) {
  const bf16x2_t v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}

typedef short s16x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 read_transposed(uint32_t at) {
  const s16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(uintptr_t)at);
  return __builtin_bit_cast(uint2, v);
}

// The state of a wave's 32 packed rows; lane l holds column l % 32, half l / 32.
template <int HD>
struct Rows {
  typedef KvTile<HD> T;
  static constexpr int kSteps = HD / 16, kChannelTiles = HD / 32, kAhead = 4, kMixAhead = HD == 256 ? 2 : 4;
  u32x4 q[kSteps];
  f32x16_t o[kChannelTiles];
  float max, sum;  // sum: this half's keys
  int pos;         // last key that the column sees, -1: none
  uint32_t places; // of the lane's operands in a tile of values (high half) and of keys

  // the columns are packed rows m0 ..
  __device__ __forceinline__ void load(const AttendArgs& a, const CutRequest& r, int kvh, int m0) {
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int m = m0 + c, in = min(m, r.packed - 1);
    const int token = (int)((uint32_t)in / (uint32_t)a.cut.group);
    const int64_t row = r.begin + token;
    const uint16_t* from = a.q + row * a.q_row + (kvh * a.cut.group + in - token * a.cut.group) * a.q_head + 8 * h;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[s] = (*reinterpret_cast<const u32x4*>(from + 16 * s) & a.q_and) ^ a.q_xor;
    pos = m < r.packed ? visible_keys(r.lead + row, r.length) - 1 : -1;
  }
  __device__ __forceinline__ void place() {
    const int lane = threadIdx.x & 63, j = lane & 15, h = lane >> 5, upper = lane >> 4 & 1;
    const int vrow = 4 * h + (j >> 2), krow = lane & 31;
    places = (uint32_t)(vrow * T::kRow + 16 * ((2 * upper + (j >> 1 & 1)) ^ T::value_swizzle(vrow)) + 8 * (j & 1)) << 16 |
             (uint32_t)(krow * T::kRow + 16 * (h ^ T::key_swizzle(krow)));
  }
  __device__ __forceinline__ void clear() {
    max = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int ct = 0; ct < kChannelTiles; ++ct) o[ct] = f32x16_t{};
  }

  // kChains running sums over the channels, added at the end: a wave alone on
  // its SIMD would otherwise wait for each product before the next.
  template <int kChains>
  __device__ __forceinline__ void scores(uint32_t keys, f32x16_t& sc) const {
    const int lane = lane_here(), row = lane & 31, h = lane >> 5;
    const uint32_t at = keys + row * T::kRow + 16 * (h ^ T::key_swizzle(row));
    auto read = [&](int s) { return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(at ^ (32 * s)); };
    // four operands on their way: more would not fit the registers beside q and o
    u32x4 k[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) k[s] = read(s);
    f32x16_t c[kChains];
#pragma unroll
    for (int i = 0; i < kChains; ++i) c[i] = f32x16_t{};
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      c[s % kChains] = mfma32(k[s % kAhead], q[s], c[s % kChains]);
      if (s + kAhead < kSteps) k[s % kAhead] = read(s + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
    sc = c[0];
#pragma unroll
    for (int i = 1; i < kChains; ++i) sc += c[i];
  }

  // Scores of N tiles to weights; `first` is the first tile's first key, `mask`
  // where some of the keys are not seen by some column (bad: two bits a tile),
  // `fresh` in front of the first product.
  template <int N>
  __device__ __forceinline__ void weights(const AttendArgs& a, f32x16_t (&t)[N], bool mask, int first, int bad, bool fresh,
                                          u32x4 (&w)[N][2]) {
    const int h = lane_here() >> 5;
    if (mask) {
      const int past = pos - first - 4 * h;  // keys beyond it are not seen
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kKeyTile * n + 8 * (r >> 2) + (r & 3) > past || (bad >> (2 * n + (r >> 3)) & 1)) t[n][r] = -INFINITY;
    }
    float most = t[0][0];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) most = fmaxf(most, t[n][r]);
    most = fmaxf(most, other_half(most)) * a.scale2;
    if (__any(most > max + kRescale)) {
      const float grown = fmaxf(max, most), keep = exp2_fast(max - (grown == -INFINITY ? 0.0f : grown));
      max = grown;
      sum *= keep;
      if (!fresh) {
#pragma unroll
        for (int ct = 0; ct < kChannelTiles; ++ct)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[ct][r] *= keep;
      }
    }
    const float base = max == -INFINITY ? 0.0f : max;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float total = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        t[n][r] = exp2_fast(__builtin_fmaf(t[n][r], a.scale2, -base));
        total += t[n][r];
      }
      sum += total;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[n][s][i] = pack_weights(t[n][8 * s + 2 * i], t[n][8 * s + 2 * i + 1]);
    }
  }

  // o += V^T P^T.
  __device__ __forceinline__ void context(uint32_t values, const u32x4 (&w)[2]) {
    const int lane = threadIdx.x & 63, j = lane & 15, h = lane >> 5, upper = lane >> 4 & 1;
    const int row = 4 * h + (j >> 2);
    const uint32_t at = values + row * T::kRow + 16 * ((2 * upper + (j >> 1 & 1)) ^ T::value_swizzle(row)) + 8 * (j & 1);
    // step n: channel tile n / 2, keys 16 (n % 2) ..
    auto read = [&](int n) {
      const uint2 x0 = read_transposed((at ^ (32 * (n & ~1))) + (16 * (n & 1)) * T::kRow);
      const uint2 x1 = read_transposed((at ^ (32 * (n & ~1))) + (16 * (n & 1) + 8) * T::kRow);
      return u32x4{x0.x, x0.y, x1.x, x1.y};
    };
    u32x4 v[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) v[n] = read(n);
#pragma unroll
    for (int n = 0; n < 2 * kChannelTiles; ++n) {
      o[n >> 1] = mfma32(v[n % kAhead], w[n & 1], o[n >> 1]);
      if (n + kAhead < 2 * kChannelTiles) v[n % kAhead] = read(n + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // o += V^T P^T and the next tile's scores in one run, product by product: the
  // scores' sum alone would have each product wait for the one before.
  __device__ __forceinline__ void mix(uint32_t values, const u32x4 (&w)[2], uint32_t keys, f32x16_t& sc) {
    uint32_t both = places;
    asm volatile("" : "+v"(both));  // taken apart here, not kept apart around the loop
    const uint32_t vat = values + (both >> 16), kat = keys + (both & 0xffff);
    auto read_value = [&](int n) {
      const uint2 x0 = read_transposed((vat ^ (32 * (n & ~1))) + (16 * (n & 1)) * T::kRow);
      const uint2 x1 = read_transposed((vat ^ (32 * (n & ~1))) + (16 * (n & 1) + 8) * T::kRow);
      return u32x4{x0.x, x0.y, x1.x, x1.y};
    };
    // steps s and s + kSteps / 2 in turn: half a row apart, their addresses differ
    // by a constant that the swizzle does not touch (256 channels)
    auto step = [](int n) { return HD == 256 ? (n >> 1) + (n & 1) * (kSteps / 2) : n; };
    auto read_key = [&](int n) {
      const uint32_t at = HD == 256 ? (kat ^ (32 * (n >> 1))) + 256 * (n & 1) : kat ^ (32 * n);
      return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)at;
    };
    constexpr int A = kMixAhead;
    u32x4 v[A], k[A];
#pragma unroll
    for (int n = 0; n < A; ++n) v[n] = read_value(n), k[n] = read_key(n);
    f32x16_t next = {};
#pragma unroll
    for (int n = 0; n < kSteps; ++n) {
      o[n >> 1] = mfma32(v[n % A], w[n & 1], o[n >> 1]);
      if (n + A < kSteps) v[n % A] = read_value(n + A);
      __builtin_amdgcn_sched_barrier(0);
      next = mfma32(k[n % A], q[step(n)], next);
      if (n + A < kSteps) k[n % A] = read_key(n + A);
      __builtin_amdgcn_sched_barrier(0);
    }
    sc = next;
  }

  // Whether a result is NaN (or infinite), also of a column that sees nothing:
  // its weights of zero meet the values that later rows see.
  __device__ __forceinline__ bool any_nan() const {
    float x = 0.0f;
#pragma unroll
    for (int ct = 0; ct < kChannelTiles; ++ct)
#pragma unroll
      for (int r = 0; r < 16; ++r) x = __builtin_fmaf(o[ct][r], 0.0f, x);
    return x != x;
  }
};

// Packed row m's results: divided by its sum, gated, rounded once; zeros for a
// row without a weight above 0, whatever its values and its gate.
struct RowWriter {
  uint16_t* out;
  const uint16_t* gate;
  float inverse;

  __device__ __forceinline__ RowWriter(const AttendArgs& a, const CutRequest& r, int kvh, int m, float sum) {
    const int token = (int)((uint32_t)m / (uint32_t)a.cut.group);
    const int64_t row = r.begin + token, head = kvh * a.cut.group + m - token * a.cut.group;
    out = a.out + row * a.out_row + head * a.out_head;
    gate = a.gate ? a.gate + row * a.gate_row + head * a.gate_head : nullptr;
    inverse = sum == 0.0f ? 0.0f : 1.0f / sum;  // 0: zeros
  }
  // Four channels from `ch` and their gates. The gates of several calls are read
  // in front of the first: behind it, each would wait for the store before it.
  __device__ __forceinline__ uint2 gates(int ch) const { return *reinterpret_cast<const uint2*>(gate + ch); }
  template <bool kGate>
  __device__ __forceinline__ void write(int ch, uint2 g, float x0, float x1, float x2, float x3) const {
    float x[4] = {x0 * inverse, x1 * inverse, x2 * inverse, x3 * inverse};
    if (kGate) {
      const float gv[4] = {lo2f(g.x), hi2f(g.x), lo2f(g.y), hi2f(g.y)};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= __builtin_amdgcn_rcpf(1.0f + exp2_fast(gv[i] * -1.44269504f));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = inverse == 0.0f ? 0.0f : x[i];
    *reinterpret_cast<uint2*>(out + ch) = make_uint2(pack_weights(x[0], x[1]), pack_weights(x[2], x[3]));
  }
};

// A partial result of 32 rows: o[channel tile][4 registers][lane] as float4,
// then 32 maxima, then 32 sums.
template <int HD>
struct PartSlot {
  static constexpr int kFloats = 32 * HD + 64;
};

// A block's item: a row tile of one KV head over one split of the keys.
struct Item {
  int request, row_tile;
  int64_t slot;
  int t0, t1;      // its key tiles
  int last_key;    // that any of its rows sees
  bool parts;      // its row tile has other splits
};

template <int kThreads>
__device__ __forceinline__ bool find_item(const AttendArgs& a, int kvh, Item* item, CutRequest* req) {
  Found f;
  if (!find_work<false, kThreads>(a, blockIdx.x / (uint32_t)a.cut.kv_heads, &f, req)) return false;
  const int splits = cut_splits(a.cut, *req, f.chunk), chunk = split_tiles(*req, splits);
  const int nth = (int)((uint32_t)f.index / (uint32_t)splits), split = f.index - nth * splits;
  item->request = f.request;
  item->row_tile = req->tiles - 1 - nth;  // the last rows, which see the most keys, first
  item->last_key = tile_keys(a.cut, *req, item->row_tile) - 1;
  const int seen = key_tiles_of(item->last_key + 1);
  item->parts = seen > chunk;
  item->t0 = split * chunk;
  item->t1 = min(item->t0 + chunk, seen);
  if (split > 0 && item->t0 >= seen) return false;
  item->slot = (f.parts_before + f.index) * a.cut.kv_heads + kvh;
  return !item->parts || item->slot < a.cut.slots;
}

// Where rows of an item came out NaN it is done again up to the least position
// among them, for the rows of that position, until none is left: a row whose own
// pass is NaN is so from what it sees. The first pass, up to the item's last key,
// writes every row that is not NaN.

// The least position among the columns of the block for which `open` holds, or
// INT32_MAX.
template <int kThreads>
__device__ __forceinline__ int least_open(bool open, int pos, int* shared) {
  int least = open ? pos : INT32_MAX;
  for (int d = 1; d < 64; d <<= 1) least = min(least, __shfl_xor(least, d, 64));
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = least;
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w) least = min(least, shared[w]);
  return __builtin_amdgcn_readfirstlane(least);
}

// ------------------------------------------------- few rows: keys over waves
//
// One item is 32 packed rows over one split of the keys; its key tiles go
// round the four waves, each with tiles of its own in LDS and no barrier until
// the end, where the waves' results are joined through LDS. A wave's next keys
// are requested when its scores are made, its next values behind the context:
// 64 KB and more are on their way per CU.
//
// Bound by the keys and values: 8 tokens over 14 to 32 thousand keys of 2 heads
// of 256, 457 MB, 90 us or 5.1 TB/s (a large copy: 4.9), and 9 us for the join.
// 512 items: one of 256 gives 125 us in all, one of 1024 (half a split each) 129.
// A single token over 520 keys is bound by its chain of loads (request, table,
// keys), 10.5 us: splits of four tiles, one a wave, against two: 20.3 and 21.3.
constexpr int kFewThreads = 256;
constexpr int kFewRows = 32;

template <int HD>
constexpr size_t few_lds_bytes() { return 4 * 2 * KvTile<HD>::kBytes; }

// An item by a block's first four waves, the others gone; kUnits: parts of a
// slot. In k_paged_many's block the scores are one chain: two spill.
template <int HD, int kUnits>
__device__ __forceinline__ void few_rows_item(const AttendArgs& a, int kvh, const Item& item, const CutRequest& req,
                                              uint8_t* lds) {
  typedef KvTile<HD> T;
  typedef Rows<HD> R;
  __shared__ float stat[2][4][32];
  __shared__ int open_at[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const int m0 = kFewRows * item.row_tile;
  const int64_t kv_offset = kvh * a.head_stride;
  R rows;
  rows.load(a, req, kvh, m0);
  // up to this key every column sees all: none where a column is no row
  const int least = m0 + kFewRows > req.packed ? -1 : visible_keys(packed_position(a.cut, req, m0), req.length) - 1;
  const uint32_t keys = lds_address(lds) + wave * 2 * T::kBytes, values = keys + T::kBytes;
  bool open = m0 + c < req.packed;  // this column's result is not written yet
  for (int limit = item.last_key;;) {
    rows.clear();
    const int t1 = min(item.t1, key_tiles_of(limit + 1)), mine = item.t0 + wave;
    Window runs;
    int window = mine;  // the window's first tile
    if (mine < t1) runs.fill(a, item.request, kv_offset, mine, 4, t1, limit);
    // tile t's keys or values
    auto request = [&](auto kind, int t) {
      constexpr bool kKeys = decltype(kind)::value;
#pragma unroll
      for (int run = 0; run < 2; ++run) {
        const int at = (t - window) / 2 + run;
        request_rows<HD, kKeys>(a, runs.at(at), runs.bad >> at & 1, 16 * run, limit - kKeyTile * t, kKeys ? keys : values, T::kLoads / 2);
      }
    };
    if (mine < t1) {
      request(std::true_type{}, mine);
      request(std::false_type{}, mine);
    }
#pragma unroll 1
    for (int t = mine; t < t1; t += 4) {
      const bool more = t + 4 < t1;
      const int gone = (int)(runs.bad >> ((t - window) / 2)) & 3;
      arrived_but<T::kLoads>();
      f32x16_t sc[1];
      rows.template scores<kUnits == 1 ? 2 : 1>(keys, sc[0]);
      __builtin_amdgcn_sched_barrier(0);
      if (more) {
        if (t + 4 == window + 128) {
          window = t + 4;
          runs.fill(a, item.request, kv_offset, window, 4, t1, limit);
        }
        request(std::true_type{}, t + 4);
      }
      u32x4 w[1][2];
      rows.template weights<1>(a, sc, kKeyTile * t + kKeyTile - 1 > least || gone, kKeyTile * t, gone, t == mine, w);
      if (more) arrived_but<T::kLoads>();
      else arrived_but<0>();
      rows.context(values, w[0]);
      __builtin_amdgcn_sched_barrier(0);
      if (more) request(std::false_type{}, t + 4);
    }
    // join the waves
    const float total = rows.sum + other_half(rows.sum);
    if (h == 0) stat[0][wave][c] = rows.max, stat[1][wave][c] = total;
    __syncthreads();
    float most = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) most = fmaxf(most, stat[0][w][c]);
    const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum += stat[1][w][c] * exp2_fast(stat[0][w][c] - base);
    const float keep = exp2_fast(rows.max - base);
    float4* red = reinterpret_cast<float4*>(lds);  // [wave][channel tile][4 registers][lane]
    constexpr int kQuads = R::kChannelTiles * 4;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const f32x16_t& o = rows.o[i >> 2];
      const int r = 4 * (i & 3);
      red[(wave * kQuads + i) * 64 + lane] = make_float4(o[r] * keep, o[r + 1] * keep, o[r + 2] * keep, o[r + 3] * keep);
    }
    __syncthreads();
    float joined[kQuads / 4][4];
    bool nan = false;
#pragma unroll
    for (int n = 0; n < kQuads / 4; ++n) {
      const int i = wave + 4 * n;
      float4 v = red[i * 64 + lane];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float4 x = red[(w * kQuads + i) * 64 + lane];
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      joined[n][0] = v.x, joined[n][1] = v.y, joined[n][2] = v.z, joined[n][3] = v.w;
      nan |= v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w;
    }
    // a column is written by all its lanes at once or not yet
    __syncthreads();
    if (lane < 32) stat[0][wave][c] = 0.0f;
    if (nan) stat[0][wave][c] = 1.0f;
    __syncthreads();
    nan = stat[0][0][c] + stat[0][1][c] + stat[0][2][c] + stat[0][3][c] != 0.0f;
    if (open && ((!nan && limit == item.last_key) || rows.pos == limit)) {
      open = false;
      if (!item.parts) {
        const RowWriter to(a, req, kvh, m0 + c, sum);
        auto write = [&](auto gate) {
          constexpr bool kGate = decltype(gate)::value;
          uint2 g[kQuads / 4] = {};
          if (kGate)
#pragma unroll
            for (int n = 0; n < kQuads / 4; ++n) g[n] = to.gates(8 * (wave + 4 * n) + 4 * h);
#pragma unroll
          for (int n = 0; n < kQuads / 4; ++n)
            to.template write<kGate>(8 * (wave + 4 * n) + 4 * h, g[n], joined[n][0], joined[n][1], joined[n][2], joined[n][3]);
        };
        if (a.gate) write(std::true_type{});
        else write(std::false_type{});
      } else {
        float* part = a.part + item.slot * kUnits * PartSlot<HD>::kFloats;
#pragma unroll
        for (int n = 0; n < kQuads / 4; ++n)
          reinterpret_cast<float4*>(part)[(wave + 4 * n) * 64 + lane] = make_float4(joined[n][0], joined[n][1], joined[n][2], joined[n][3]);
        if (wave == 0 && h == 0) part[32 * HD + c] = most, part[32 * HD + 32 + c] = sum;
      }
    }
    limit = least_open<kFewThreads>(open, rows.pos, open_at);
    if (limit == INT32_MAX) break;
    __syncthreads();
  }
}

template <int HD>
__global__ __launch_bounds__(kFewThreads, HD == 256 ? 1 : 2) void k_paged_few(AttendArgs a) {
  extern __shared__ __align__(1024) uint8_t attend_lds[];
  const int kvh = blockIdx.x % (uint32_t)a.cut.kv_heads;
  Item item;
  CutRequest req;
  if (find_item<kFewThreads>(a, kvh, &item, &req)) few_rows_item<HD, 1>(a, kvh, item, req, attend_lds);
}

// -------------------------------------------- many rows: rows over waves
//
// One item is 256 packed rows over one split of the keys, 32 rows a wave, two
// waves a SIMD. The waves share rings of four stages of 32 keys (of 64 for heads
// of up to 128 channels, whose tiles are short), half of them requesting the
// keys, half the values, two to three stages ahead; one barrier a stage. A
// request of up to 32 packed rows is done as in k_paged_few.
//
// A stage is its softmax on the vector unit and a run of products (its values',
// the next stage's scores) on the matrix cores. The first half of the waves
// enters a stage in front of its softmax, the second, on the same SIMDs, in
// front of the products of the stage before, so that one's softmax meets the
// other's products. No register of a lane is left at 256 channels (q 64, o 128,
// scores 16, weights 8, operands under way 16): what can be made anew in the
// loop is, since a spilled register's reload waits for all requests.
//
// Bound by power: 2048 tokens of 16 heads over 32768 keys of 2 heads of 256 take
// 0.99 ms, 1.08 PFLOP/s (a large product: 1.2), the matrix cores busy half of the
// cycles of a clock that falls from 2.3 to 1.8 - 2.0 GHz. In step, scores in a
// run of their own: 1.08 ms; a phase apart with that run: 1.15 ms; values'
// products and scores in one run without places in the lanes (table and strides
// worked on every stage): 1.26 ms. 16 mixed requests (500, 300, 223 and single
// tokens over up to 4096 keys of 256 channels) take 59 to 62 us, 18 more for the
// join: 19 stages, then 44 MB of partial results by all items at once.
constexpr int kManyThreads = 512;
constexpr int kManyRows = 256;
constexpr int kManyStages = 4;
template <int HD>
constexpr int kStageTiles = HD == 256 ? 1 : 2;

template <int HD>
constexpr size_t many_lds_bytes() { return kManyStages * kStageTiles<HD> * 2 * KvTile<HD>::kBytes; }

template <int HD>
__global__ __launch_bounds__(kManyThreads, 2) void k_paged_many(AttendArgs a) {
  typedef KvTile<HD> T;
  typedef Rows<HD> R;
  constexpr int N = kStageTiles<HD>;
  extern __shared__ __align__(1024) uint8_t attend_lds[];
  __shared__ int open_at[8];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const int kvh = blockIdx.x % (uint32_t)a.cut.kv_heads;
  Item item;
  CutRequest req;
  if (!find_item<kManyThreads>(a, kvh, &item, &req)) return;
  if (req.packed <= kFewRows) {
    if (wave < kFewThreads / 64) few_rows_item<HD, kManyRows / 32>(a, kvh, item, req, attend_lds);
    return;
  }
  const int m0 = kManyRows * item.row_tile + 32 * wave;
  const int64_t kv_offset = kvh * a.head_stride;
  R rows;
  const int least = m0 + 32 > req.packed ? -1 : visible_keys(packed_position(a.cut, req, m0), req.length) - 1;
  const bool idle = m0 >= req.packed;  // no rows: the wave only requests tiles
  const bool late = wave >= 4;
  const uint32_t key_ring = lds_address(attend_lds), value_ring = key_ring + kManyStages * N * T::kBytes;
  // The first four waves request a stage's keys, the others its values; a
  // wave's share is of one run of 16 rows (half a run for 256 channels).
  constexpr int kOwn = N * T::kLoads / 4;
  const int share = (wave & 3) * kOwn, own_tile = share / T::kLoads, own_row = share % T::kLoads * T::kPer;
  const int own_run = 2 * own_tile + (own_row >> 4);
  bool open = m0 + c < req.packed;
  for (int limit = item.last_key;;) {
    rows.load(a, req, kvh, m0);  // again with each pass: not kept over the results' writing
    rows.clear();
    const int t1 = min(item.t1, key_tiles_of(limit + 1)), stages = (t1 - item.t0 + N - 1) / N;
    Window runs;
    uint64_t bad_before = 0;  // of the window before
    auto request = [&](int i) {
      const int run = 2 * N * i & 63;
      if (run == 0) {
        bad_before = i > 0 ? runs.bad : 0;
        runs.fill(a, item.request, kv_offset, item.t0 + N * i, 1, t1, limit);
      }
      const bool bad = runs.bad >> (run + own_run) & 1;
      const int last = limit - kKeyTile * (item.t0 + N * i + own_tile);
      const uint32_t slot = (uint32_t)(i % kManyStages * N + own_tile) * T::kBytes;
      if (late) request_rows<HD, false>(a, runs.at(run + own_run), bad, own_row, last, value_ring + slot, kOwn);
      else request_rows<HD, true>(a, runs.at(run + own_run), bad, own_row, last, key_ring + slot, kOwn);
    };
    // the bad runs of stage i; the window may be a later one's by then
    const int ahead = late ? 2 : 3;
    auto bad_runs = [&](int i) {
      const int newest = min(i + ahead, stages - 1);  // requested by now
      const uint64_t b = (2 * N * newest) / 64 == (2 * N * i) / 64 ? runs.bad : bad_before;
      return (int)(b >> (2 * N * i & 63)) & ((1 << 2 * N) - 1);
    };
#pragma unroll 1
    for (int i = 0; i < ahead; ++i)
      if (i < stages) request(i);
    // Barrier i: the keys of stage i + 1 and the values of stage i are in LDS
    // for every wave, the keys of stage i - 1 and the values of stage i - 2 done
    // with.
    auto enter = [&](int i) {
      if (i + ahead - 1 < stages) arrived_but<kOwn>();
      else arrived_but<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");  // no LDS read of the stages in front of it
      __builtin_amdgcn_sched_barrier(0);
      if (i + ahead < stages) request(i + ahead);
    };
    auto keys_at = [&](int i) { return key_ring + (uint32_t)(i % kManyStages * N) * T::kBytes; };
    auto values_at = [&](int i) { return value_ring + (uint32_t)(i % kManyStages * N) * T::kBytes; };
    rows.place();
    if (stages <= 0) {  // no key is seen
    } else if (idle) {
#pragma unroll 1
      for (int i = 0; i <= stages; ++i) enter(i);
    } else {
      f32x16_t sc[N];
      enter(0);
#pragma unroll
      for (int n = 0; n < N; ++n) rows.template scores<1>(keys_at(0) + n * T::kBytes, sc[n]);
#pragma unroll 1
      for (int i = 0; i < stages; ++i) {
        if (!late && i > 0) enter(i);
        const int gone = bad_runs(i), first = kKeyTile * (item.t0 + N * i);
        u32x4 w[N][2];
        rows.template weights<N>(a, sc, first + kKeyTile * N - 1 > least || gone, first, gone, i == 0, w);
        __builtin_amdgcn_sched_barrier(0);
        if (late) enter(i + 1);
        // behind the last stage the scores are of what the ring held: not used
#pragma unroll
        for (int n = 0; n < N; ++n) rows.mix(values_at(i) + n * T::kBytes, w[n], keys_at(i + 1) + n * T::kBytes, sc[n]);
      }
      if (!late) enter(stages);
    }
    __syncthreads();
    // keys that every row sees are no reason to do a row again
    const bool whole = kKeyTile * item.t1 <= visible_keys(packed_position(a.cut, req, kManyRows * item.row_tile), req.length);
    bool nan = !whole && rows.any_nan();
    nan |= __shfl_xor((int)nan, 32, 64) != 0;
    const float sum = rows.sum + other_half(rows.sum);
    if (open && ((!nan && limit == item.last_key) || rows.pos == limit)) {
      open = false;
      if (!item.parts) {
        const RowWriter to(a, req, kvh, m0 + c, sum);
        auto write = [&](auto gate) {
          constexpr bool kGate = decltype(gate)::value;
          constexpr int kBatch = 8;
#pragma unroll
          for (int i0 = 0; i0 < R::kChannelTiles * 4; i0 += kBatch) {
            uint2 g[kBatch] = {};
            if (kGate)
#pragma unroll
              for (int n = 0; n < kBatch; ++n) g[n] = to.gates(8 * (i0 + n) + 4 * h);
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
              const f32x16_t& o = rows.o[(i0 + n) >> 2];
              const int r = 4 * (n & 3);
              to.template write<kGate>(8 * (i0 + n) + 4 * h, g[n], o[r], o[r + 1], o[r + 2], o[r + 3]);
            }
          }
        };
        if (a.gate) write(std::true_type{});
        else write(std::false_type{});
      } else {
        // the addresses made here: kept over the loop they are spilled, and each
        // reload waits for the stores in front of it
        float* part = a.part + (item.slot * (kManyRows / 32) + wave) * PartSlot<HD>::kFloats;
        const uint32_t own = 4 * lane_here();
#pragma unroll
        for (int i = 0; i < R::kChannelTiles * 4; ++i) {
          const f32x16_t& o = rows.o[i >> 2];
          const int r = 4 * (i & 3);
          *reinterpret_cast<float4*>(part + 256 * i + own) = make_float4(o[r], o[r + 1], o[r + 2], o[r + 3]);
        }
        if (h == 0) part[32 * HD + c] = rows.max, part[32 * HD + 32 + c] = sum;
      }
    }
    limit = least_open<kManyThreads>(open, rows.pos, open_at);
    if (limit == INT32_MAX) break;
    __syncthreads();
  }
}

// ---------------------------------------------------- joining the splits
//
// Block (32 packed rows and KV head, kTiles channel tiles): each thread a
// float4 of the fragment order per channel tile over all splits, or over those
// of its group of four waves, weighted by 2^(max - maximum). The splits' maxima
// and sums are read once, two a wave at a time, each wave's joined as they come;
// the first parts and the gate are on their way meanwhile.
template <int HD, int kUnits, int kTiles, int kGroups>
__global__ __launch_bounds__(256 * kGroups) void k_paged_join(AttendArgs a) {
  static_assert(kGroups == 1 || kTiles == 1, "groups are added once");
  constexpr int kWaves = 4 * kGroups, kJoinKept = kGroups > 1 ? 256 : 128;  // splits whose maxima stay in LDS
  const int kvh = blockIdx.x % (uint32_t)a.cut.kv_heads;
  const uint32_t unit = blockIdx.x / (uint32_t)a.cut.kv_heads;
  Found f;
  CutRequest req;
  if (!find_work<true, 256 * kGroups>(a, unit / kUnits, &f, &req)) return;
  const int splits = cut_splits(a.cut, req, f.chunk), chunk = split_tiles(req, splits);
  const int tile = req.tiles - 1 - f.index, seen = key_tiles_of(tile_keys(a.cut, req, tile));
  if (seen <= chunk) return;
  const int used = (int)((uint32_t)(seen + chunk - 1) / (uint32_t)chunk), of = (int)(unit % kUnits);
  const int64_t first = (f.parts_before + (int64_t)f.index * splits) * a.cut.kv_heads + kvh;
  if (first + (int64_t)(used - 1) * a.cut.kv_heads >= a.cut.slots) return;
  __shared__ float kept[kJoinKept][32], stat[2][2 * kWaves][32];
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = kGroups > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : threadIdx.x >> 6;
  const int m0 = a.cut.tile_rows * tile + 32 * of, m = min(m0 + c, req.packed - 1);
  if (m0 >= req.packed) return;
  const bool row = m0 + c < req.packed;  // other columns' parts were not written
  const int64_t step = (int64_t)a.cut.kv_heads * kUnits * PartSlot<HD>::kFloats;
  const float* part = a.part + (first * kUnits + of) * PartSlot<HD>::kFloats;
  const int quad0 = 4 * kTiles * blockIdx.y + (kGroups > 1 ? wave & 3 : wave);  // this thread's quads: quad0 + 4 j
  RowWriter to(a, req, kvh, m, 1.0f);
  const int each = (used + kGroups - 1) / kGroups;
  const int begin = kGroups > 1 ? wave / 4 * each : 0, end = kGroups > 1 ? min(begin + each, used) : used;
  constexpr int kBatch = 8;
  float4 x[kBatch];
  auto read = [&](int s0, int j) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      x[i] = s0 + i < end && row ? reinterpret_cast<const float4*>(part + (s0 + i) * step)[(quad0 + 4 * j) * 64 + lane]
                                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  };
  read(begin, 0);
  uint2 g[kTiles] = {};
  if (a.gate)
#pragma unroll
    for (int j = 0; j < kTiles; ++j) g[j] = to.gates(8 * (quad0 + 4 * j) + 4 * h);
  float most = -INFINITY, sum = 0.0f;
  if (row)
#pragma unroll 4
    for (int s = 2 * wave + h; s < used; s += 2 * kWaves) {
      const float x = part[s * step + 32 * HD + c], l = part[s * step + 32 * HD + 32 + c];
      if (s < kJoinKept) kept[s][c] = x;
      const float grown = fmaxf(most, x), base = grown == -INFINITY ? 0.0f : grown;
      sum = __builtin_fmaf(l, exp2_fast(x - base), sum * exp2_fast(most - base));
      most = grown;
    }
  stat[0][2 * wave + h][c] = most, stat[1][2 * wave + h][c] = sum;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2 * kWaves; ++i) most = fmaxf(most, stat[0][i][c]);
  const float base = most == -INFINITY ? 0.0f : most;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 2 * kWaves; ++i) sum = __builtin_fmaf(stat[1][i][c], exp2_fast(stat[0][i][c] - base), sum);
  const float inverse = 1.0f / sum;
  if (sum == 0.0f) to.inverse = 0.0f;
#pragma unroll
  for (int j = 0; j < kTiles; ++j) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = begin; s0 < end; s0 += kBatch) {
      if (s0 > begin || j > 0) read(s0, j);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int s = s0 + i;
        if (s >= end) break;
        const float w = exp2_fast((s < kJoinKept ? kept[s][c] : part[s * step + 32 * HD + c]) - base) * inverse;
        v.x = __builtin_fmaf(w, x[i].x, v.x), v.y = __builtin_fmaf(w, x[i].y, v.y);
        v.z = __builtin_fmaf(w, x[i].z, v.z), v.w = __builtin_fmaf(w, x[i].w, v.w);
      }
    }
    if (kGroups > 1) {
      __shared__ float4 sums[kGroups][4][64];
      sums[wave / 4][wave & 3][lane] = v;
      __syncthreads();
      if (wave >= 4) return;
#pragma unroll
      for (int o = 1; o < kGroups; ++o) {
        const float4 y = sums[o][wave][lane];
        v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
      }
    }
    if (!row) continue;
    if (a.gate) to.template write<true>(8 * (quad0 + 4 * j) + 4 * h, g[j], v.x, v.y, v.z, v.w);
    else to.template write<false>(8 * (quad0 + 4 * j) + 4 * h, g[j], v.x, v.y, v.z, v.w);
  }
}

// ------------------------------------------------------------- host side

// How a call of paged attention is cut. k_paged_few reads the keys again for
// every 32 packed rows (rows times query heads of a KV head), k_paged_many for
// every 256, but its items are longer and have more to write. Requests of up to
// 32 packed rows, and calls whose 32-row tiles of a KV head times keys times
// channels stay below kFewWork, go to the first. Measured in us, few and many,
// at tiles x keys: 256 channels 512 x 600 45, 46; 64 x 4000 42, 42; 128 x 4000
// 56, 55; 1024 x 600 81, 60; 256 x 4000 91, 73; 64 x 16000 84, 70. 128 channels
// 256 x 4000 40, 44; 512 x 4000 61, 59; 256 x 16000 115, 93. 64 channels 2048 x
// 600 31, 38; 512 x 4000 46, 44; 256 x 16000 84, 67. max_rows and max_keys tell
// without the lengths, a call without max_keys counts as one of kKeysAssumed;
// max_keys also spares the join where no request can be split.
constexpr int64_t kFewWork = 1 << 27;
constexpr int64_t kKeysAssumed = 4096;
constexpr int kFewTarget = 9, kManyTarget = 8;  // log2 of the items wanted
constexpr int kFewMinTiles = 4, kManyMinTiles = 8;
constexpr int kMostSplits = 1024;
constexpr int64_t kMostBlocks = 1 << 22;  // times 512 threads: a launch takes below 2^32
// Few units take a channel tile a block, and four groups of waves where a row
// tile may have kTallJoin splits, a chain of loads for one (one token over 32768 keys
// of 2 heads of 256 in 256 splits: 48 and 84 us; over 8000 20 and 27); 32 requests
// of 5 over 5000, of five splits, 66 and 57.5.
constexpr int kWideJoin = 512;  // units of 32 packed rows and KV head

struct AttendPlan {
  bool few, tall;        // tall: row tiles of many splits
  CutRule cut;
  int64_t items, units;  // at most: blocks of the attention, 32-row groups of the join
  int64_t floats;        // of workspace
};

inline AttendPlan cut_attention(bool few, int64_t rows, int64_t requests, int q_heads, int kv_heads, int head_dim,
                                int64_t max_keys) {
  AttendPlan p{};
  const int group = q_heads / kv_heads;
  p.few = few;
  CutRule& c = p.cut;
  c.rows = (int32_t)rows, c.group = group, c.kv_heads = kv_heads, c.tile_rows = p.few ? kFewRows : kManyRows;
  c.target_shift = p.few ? kFewTarget : kManyTarget, c.min_tiles = p.few ? kFewMinTiles : kManyMinTiles;
  c.search = !p.few;
  const int64_t key_tiles = max_keys > 0 ? (std::min<int64_t>(max_keys, INT32_MAX) + kKeyTile - 1) / kKeyTile : INT32_MAX;
  c.max_splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>(kMostSplits, (key_tiles + c.min_tiles - 1) / c.min_tiles));
  const int64_t tiles = most_tiles(rows, requests, group, c.tile_rows);
  p.items = most_items(tiles, kv_heads, c.target_shift, c.max_splits);
  p.units = tiles * kv_heads * (c.tile_rows / 32);
  c.slots = most_slots(tiles, kv_heads, c.target_shift, c.max_splits);
  p.tall = c.slots >= kTallJoin * tiles * kv_heads;
  p.floats = c.slots * (c.tile_rows / 32) * (32 * (int64_t)head_dim + 64);
  return p;
}

inline AttendPlan plan_attention(int64_t rows, int64_t requests, int q_heads, int kv_heads, int head_dim, int64_t max_rows,
                                 int64_t max_keys) {
  const int64_t group = q_heads / kv_heads, longest = (max_rows > 0 ? std::min(max_rows, rows) : rows) * group;
  const int64_t tiles = rows * group / kFewRows * kv_heads, keys = max_keys > 0 ? max_keys : kKeysAssumed;
  return cut_attention(longest <= kFewRows || tiles <= kFewWork / head_dim / keys, rows, requests, q_heads, kv_heads, head_dim,
                       max_keys);
}

// The most floats of workspace that one request of up to `rows` rows and
// `max_keys` keys asks for.
inline int64_t most_attend_floats(int64_t rows, int q_heads, int kv_heads, int head_dim, int64_t max_keys) {
  return std::max(cut_attention(true, rows, 1, q_heads, kv_heads, head_dim, max_keys).floats,
                  cut_attention(false, rows, 1, q_heads, kv_heads, head_dim, max_keys).floats);
}

struct AttendKernels {
  void (*attend)(AttendArgs);
  void (*join)(AttendArgs);
  dim3 grid, join_grid;
  int threads, join_threads;
  size_t lds;
};

template <int HD>
AttendKernels attend_kernels(const AttendPlan& p) {
  // a block a channel tile where there are few rows, all of them where there are many
  const bool wide = p.units >= kWideJoin;
  AttendKernels k;
  k.attend = p.few ? k_paged_few<HD> : k_paged_many<HD>;
  constexpr int kUnits = kManyRows / 32;
  const bool tall = !wide && p.tall;
  k.join = p.few ? (wide ? k_paged_join<HD, 1, HD / 32, 1> : tall ? k_paged_join<HD, 1, 1, 4> : k_paged_join<HD, 1, 1, 1>)
                 : (wide ? k_paged_join<HD, kUnits, HD / 32, 1> : tall ? k_paged_join<HD, kUnits, 1, 4> : k_paged_join<HD, kUnits, 1, 1>);
  k.join_threads = tall ? 1024 : 256;
  k.grid = dim3((unsigned)p.items), k.join_grid = dim3((unsigned)p.units, wide ? 1 : HD / 32);
  k.threads = p.few ? kFewThreads : kManyThreads;
  k.lds = p.few ? few_lds_bytes<HD>() : many_lds_bytes<HD>();
  return k;
}

inline void attend_scale(AttendArgs* a, float scale) {
  a->scale2 = scale == 0.0f ? 1.0f : (scale < 0.0f ? -scale : scale) * 1.44269504f;
  a->q_and = scale == 0.0f ? 0u : ~0u, a->q_xor = scale < 0.0f ? 0x80008000u : 0u;
}

// A request over a contiguous cache: its rows, length and a table of pages
// that follow each other, for attention over the session's own cache. A chunk of
// a prompt is a request for every kSpanRows of its rows, attended by a call of
// its own: how a call is cut, and so its rounding, follows from its rows, and
// chunks of any whole number of kSpanRows (fewer rows are taken where memory is
// short) then give the same bits.
constexpr int kSpanShift = 16, kSpanTable = 64;  // rows of a page (log2), pages
constexpr int kSpanRows = 1024;
struct PromptSpan {
  int32_t row_start[2], length, pad;
  int32_t table[kSpanTable];
};
__global__ void k_prompt_span(const uint64_t* __restrict__ params, int t, int rows_n, PromptSpan* __restrict__ spans) {
  const int i = threadIdx.x, before = kSpanRows * blockIdx.x, rows = min(kSpanRows, rows_n - before);
  PromptSpan* span = spans + blockIdx.x;
  if (i < kSpanTable) span->table[i] = i;
  if (i == 0) {
    span->row_start[0] = 0, span->row_start[1] = rows;
    span->length = (int32_t)(step_position(params, t) + before + rows);
  }
}

}  // namespace cq35
