// Index arithmetic of the paged-cache operators: plain C++ for the device and
// the host (the CPU tests compile it with the host compiler).
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define CQ35_BOTH __host__ __device__ inline
#else
#define CQ35_BOTH inline
#endif

namespace cq35 {

// Pages that hold `tokens` tokens (a power-of-two page: 1 << shift rows).
CQ35_BOTH int64_t pages_of(int64_t tokens, int shift) { return (tokens + (1 << shift) - 1) >> shift; }

// The last request whose first row is at or before `row` (starts ascending,
// starts[0] <= row): requests without rows in front of it are passed over.
CQ35_BOTH int request_of(const int32_t* starts, int requests, int64_t row) {
  int lo = 0, hi = requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// What a page plan makes of one request: the rows it appends, the pages it
// takes and the pages it gives back.
struct PlanNeed {
  int64_t rows, take, give;
  bool bad;
};
CQ35_BOTH PlanNeed plan_need(int64_t cached, int64_t length, int64_t width, int shift) {
  const int64_t have = pages_of(cached, shift), want = pages_of(length, shift);
  if (cached < 0 || length < 0 || have > width || want > width) return {0, 0, 0, true};
  return {length > cached ? length - cached : 0, want > have ? want - have : 0, have > want ? have - want : 0, false};
}

// The outcome of a plan from its totals.
enum PlanCode { kPlanOk = 0, kPlanPages = 1, kPlanRows = 2, kPlanLengths = 3, kPlanStack = 4 };
struct PlanVerdict {
  int32_t code;
  int64_t missing;  // pages or rows too few
};
CQ35_BOTH PlanVerdict plan_verdict(bool bad, int64_t free_pages, int64_t pages, int64_t rows_total, int64_t take,
                                   int64_t give, int64_t rows) {
  if (bad) return {kPlanLengths, 0};
  if (free_pages < 0 || free_pages + give > pages) return {kPlanStack, 0};
  if (rows_total > rows) return {kPlanRows, rows_total - rows};
  if (take > free_pages + give) return {kPlanPages, take - free_pages - give};
  return {kPlanOk, 0};
}

// Cache row of position p of a page: page * rows + p % rows, -1 for a page
// number outside the cache.
CQ35_BOTH int32_t slot_of(int32_t page, int64_t pages, int64_t position, int shift) {
  if (page < 0 || page >= pages) return -1;
  return (int32_t)(((int64_t)page << shift) + (position & ((1 << shift) - 1)));
}

// ------------------------------------------------- how attention is cut
//
// A request's packed rows (row * group + query head of its KV head) are dealt
// in tiles of `tile_rows`; the keys a tile sees are dealt in tiles of kKeyTile
// and those in splits of equal length. How long a split is follows from all
// requests' (row tile, key tile) pairs over the number of items wanted, so
// that few rows over many keys fill the chip and many rows are not split.
constexpr int kKeyTile = 32;

struct CutRule {
  int32_t rows;         // of q; rows * group is below 2^31
  int32_t most_keys;    // that a table row holds
  int32_t group, kv_heads, tile_rows;
  int32_t target_shift; // log2 of the items wanted, over all KV heads
  int32_t min_tiles;    // key tiles of a split at least
  int32_t max_splits;
  int32_t search;       // up to 64 requests: look for the chunk of the fewest rounds
  int64_t slots;        // partial results that the workspace holds
};

struct CutRequest {
  int32_t begin, end;  // rows inside q
  int64_t lead;        // position of row t: lead + t
  int32_t length;
  int32_t packed, tiles;
  int32_t key_tiles;   // that its last row sees
};

CQ35_BOTH int32_t visible_keys(int64_t position, int32_t length) {
  return position < 0 ? 0 : position + 1 < length ? (int32_t)(position + 1) : length;
}
CQ35_BOTH int32_t key_tiles_of(int32_t keys) { return (int32_t)(((uint32_t)keys + kKeyTile - 1) / kKeyTile); }

CQ35_BOTH CutRequest cut_request(const CutRule& c, int32_t start, int32_t stop, int32_t length) {
  CutRequest q;
  q.begin = start < 0 ? 0 : start;
  q.end = stop < c.rows ? stop : c.rows;
  q.length = length < 0 ? 0 : length < c.most_keys ? length : c.most_keys;
  q.lead = (int64_t)q.length - stop;
  q.packed = q.end > q.begin ? (q.end - q.begin) * c.group : 0;
  q.tiles = (int32_t)(((uint32_t)q.packed + c.tile_rows - 1) / (uint32_t)c.tile_rows);
  q.key_tiles = q.packed ? key_tiles_of(visible_keys(q.lead + q.end - 1, q.length)) : 0;
  return q;
}

// Where row tiles are of more rows, a request of up to kLightRows packed rows is
// dealt with by four waves, a key tile each, in about half the time a tile of
// the others takes: its splits are kLightTimes as long (500, 300, 223 rows and 13
// single tokens, 256 channels: 79.8 us, at three times 80, with splits and waves
// as for the others 85.4).
constexpr int kLightRows = 32, kLightTimes = 2;
CQ35_BOTH int32_t key_weight(const CutRule& c, const CutRequest& q) {
  return c.tile_rows > kLightRows && q.packed <= kLightRows ? kLightTimes : 1;
}
CQ35_BOTH int64_t request_work(const CutRule& c, const CutRequest& q) {
  const int32_t w = key_weight(c, q);
  return ((int64_t)q.tiles * q.key_tiles + w - 1) / w;
}

// Splits of a request's row tiles, and the key tiles of each.
CQ35_BOTH int32_t cut_splits(const CutRule& c, const CutRequest& q, int32_t chunk) {
  chunk *= key_weight(c, q);
  if (q.key_tiles <= chunk) return 1;
  const int32_t n = (int32_t)(((uint32_t)q.key_tiles + chunk - 1) / (uint32_t)chunk);
  return n < c.max_splits ? n : c.max_splits;
}
CQ35_BOTH int32_t split_tiles(const CutRequest& q, int32_t splits) {
  return q.key_tiles ? (int32_t)(((uint32_t)q.key_tiles + splits - 1) / (uint32_t)splits) : 1;
}

// Key tiles of a split, from the sum of the requests' work (tiles * key_tiles):
// that sum dealt evenly to the items wanted, or up to twice that (`search`)
// where the requests' ends then make fewer rounds of items: one CU holds one,
// and an item costs some tiles' time besides its own (kItemTiles, measured).
// Tiles of few rows that may have many splits take up to twice min_tiles first,
// half as many items as wanted: one token over 32768 keys of 2 heads of 256 33
// us, with twice the splits 47 (2 requests of 3 over 17909 keys of one head 26
// and 36).
// items_at(chunk): the items per KV head that splits of `chunk` make.
constexpr int kItemTiles = 6;
constexpr int kTallJoin = 32;  // splits of a row tile from which on its join is a chain
template <typename F>
CQ35_BOTH int32_t cut_chunk(const CutRule& c, int64_t pairs, F items_at) {
  const int64_t even = (pairs * c.kv_heads + ((int64_t)1 << c.target_shift) - 1) >> c.target_shift;
  const int64_t twice = 2 * even < 2 * c.min_tiles ? 2 * even : 2 * c.min_tiles;
  const int64_t least_tiles = c.tile_rows <= kLightRows && c.max_splits >= kTallJoin && twice > c.min_tiles ? twice : c.min_tiles;
  const int64_t wanted = even > least_tiles ? even : least_tiles;
  const int32_t base = wanted > INT32_MAX / 16 ? INT32_MAX / 16 : (int32_t)wanted;
  if (!c.search) return base;
  int32_t best = base;
  int64_t least = INT64_MAX;
  for (int k = 0; k < 5; ++k) {
    const int32_t chunk = base + (base >> 2) * k;
    const int64_t rounds = (items_at(chunk) * c.kv_heads + ((int64_t)1 << c.target_shift) - 1) >> c.target_shift;
    const int64_t cost = rounds * (chunk + kItemTiles);
    if (cost < least) least = cost, best = chunk;
  }
  return best;
}

// Position of packed row m of a request.
CQ35_BOTH int64_t packed_position(const CutRule& c, const CutRequest& q, int32_t m) {
  return q.lead + q.begin + (int32_t)((uint32_t)m / (uint32_t)c.group);
}
// Keys that row tile i of a request sees (its last row's).
CQ35_BOTH int32_t tile_keys(const CutRule& c, const CutRequest& q, int32_t i) {
  const int64_t past = (int64_t)(i + 1) * c.tile_rows;
  return visible_keys(packed_position(c, q, (int32_t)(past < q.packed ? past : q.packed) - 1), q.length);
}

// Bounds that hold for any lengths: row tiles per KV head of a launch over
// `rows` rows of `requests` requests, items over all KV heads (a split row tile
// has at most 1 + its share of the work / chunk of them, and the work / chunk is
// at most target / kv_heads), partial results (at most twice that, as only
// tiles of two splits or more have any).
CQ35_BOTH int64_t most_tiles(int64_t rows, int64_t requests, int group, int tile_rows) {
  return rows * group / tile_rows + (rows < requests ? rows : requests);
}
CQ35_BOTH int64_t most_items(int64_t tiles, int kv_heads, int target_shift, int max_splits) {
  const int64_t a = tiles + ((int64_t)1 << target_shift) / kv_heads, b = tiles * max_splits;
  return (a < b ? a : b) * kv_heads;
}
CQ35_BOTH int64_t most_slots(int64_t tiles, int kv_heads, int target_shift, int max_splits) {
  if (max_splits == 1) return 0;
  const int64_t a = (int64_t)2 << target_shift, b = tiles * max_splits * kv_heads;
  return a < b ? a : b;
}

}  // namespace cq35
