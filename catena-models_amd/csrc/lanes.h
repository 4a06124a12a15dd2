// Sums and maxima over the lanes of a wave, the result in every lane and of the same bits there:
// neighbours by data-parallel moves inside rows of 16, then the rows of 16 and of 32
// swapped. About a dozen instructions; a shuffle through LDS takes as long for each of its six steps.
#pragma once

#include <hip/hip_runtime.h>

namespace cq35 {

template <int kCtrl, typename T>
__device__ __forceinline__ T lane_moved(T x) {
  const int i = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(i, i, kCtrl, 0xf, 0xf, false));
}

// x and the other half's of each pair of rows of 16, or of the two of 32, in an order that both share.
struct LanePair {
  int a, b;
};
__device__ __forceinline__ LanePair rows16_pair(int x) {
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return {(int)r[0], (int)r[1]};
}
__device__ __forceinline__ LanePair rows32_pair(int x) {
  const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return {(int)r[0], (int)r[1]};
}

// f is commutative; every lane active.
template <typename T, typename F>
__device__ __forceinline__ T over_lanes(T x, F f) {
  x = f(x, lane_moved<0xb1>(x));   // lane ^ 1
  x = f(x, lane_moved<0x4e>(x));   // lane ^ 2
  x = f(x, lane_moved<0x141>(x));  // the other quad of 8
  x = f(x, lane_moved<0x140>(x));  // the other 8 of 16
  const LanePair r = rows16_pair(__builtin_bit_cast(int, x));
  x = f(__builtin_bit_cast(T, r.a), __builtin_bit_cast(T, r.b));
  const LanePair h = rows32_pair(__builtin_bit_cast(int, x));
  return f(__builtin_bit_cast(T, h.a), __builtin_bit_cast(T, h.b));
}

__device__ __forceinline__ float lanes_sum(float x) {
  return over_lanes(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float lanes_max(float x) {
  return over_lanes(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
  return over_lanes(x, [](uint32_t a, uint32_t b) { return max(a, b); });
}

}  // namespace cq35
