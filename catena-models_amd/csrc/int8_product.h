// Product of 8-bit rows: out[m][n] = (sum_k x[m][k] w[n][k]) sx[m] sw[n], the sums
// exact in 32-bit integers (channels <= 2^16, so they stay below 2^30), the two
// products and the rounding of the sum to F32 one rounding each, the result rounded once
// more where it is BF16.
#pragma once

#include "layers.h"

namespace cq35 {

constexpr int kProductMostChannels = 1 << 16;

struct ProductArgs {
  const int8_t *x, *w;
  int64_t x_stride, w_stride;
  const float *sx, *sw;
  int64_t rows, outputs;
  int channels;
  void* out;
  int64_t out_stride;
};

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ void store_product(float v, uint16_t* to) { *to = f2bf(v); }
__device__ __forceinline__ void store_product(float v, float* to) { *to = v; }

// Block = 64 rows x 64 outputs, a wave 32 x 32 of them. Weights are the first operand of the
// matrix instruction, so that a lane's results are four outputs of one row.
template <typename T>
__global__ __launch_bounds__(256) void k_int8_product(ProductArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const uint32_t across = (uint32_t)((a.outputs + 63) / 64);
  const int64_t m = (int64_t)(blockIdx.x / across) * 64 + 32 * (wave & 1) + c, n0 = (int64_t)(blockIdx.x % across) * 64 + 32 * (wave >> 1);
  const int8_t* x = a.x + min(m, a.rows - 1) * a.x_stride;
  const int8_t* w = a.w + min(n0 + c, a.outputs - 1) * a.w_stride;
  i32x16 acc = {};
  for (int k = 16 * h; k < a.channels + 16 * h; k += 32) {
    const i32x4 zero = {};
    const bool in = k < a.channels;
    const i32x4 wv = in ? *reinterpret_cast<const i32x4*>(w + k) : zero, xv = in ? *reinterpret_cast<const i32x4*>(x + k) : zero;
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(wv, xv, acc, 0, 0, 0);
  }
  if (m >= a.rows) return;
  const float sx = a.sx[m];
  T* out = (T*)a.out + m * a.out_stride;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t n = n0 + 8 * (i >> 2) + 4 * h + (i & 3);
    if (n < a.outputs) store_product((float)acc[i] * sx * a.sw[n], out + n);
  }
}

}  // namespace cq35
