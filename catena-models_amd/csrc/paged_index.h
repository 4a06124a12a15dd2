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

}  // namespace cq35
