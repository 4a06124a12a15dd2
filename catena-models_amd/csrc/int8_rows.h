// Rows of 8-bit integers with a scale each: plain rows (k_int8_rows of
// RowSource::kPlain), the norm of rows with the residual's addition
// (RowSource::kNorm) and the gated product of a feed-forward (RowSource::kGated).
//
// One pass: a row stays in registers between its sums and its integers. Bound by bytes where there are
// many rows: 8192 rows of 4096 channels 21.7 us (4.7 TB/s; a large copy: 5.0), of 2048 with residual and
// norm 26.2 (4.5), of 6144 gated 49.9 (5.0); where results go to the same memory each time 19.2, 22.9 and 45.5. A
// row or a few are latency, 2.4 to 4 us. With the norm's weights read for every row behind its sum, and no next row
// under way, the second took 30 us. Rows beyond 8192 channels: 4096 of 12288 normed with residual 86 us (4.1 TB/s;
// F32 145, 4.5), gated 67 (3.8; F32 93, 4.9).
#pragma once

#include "lanes.h"
#include "layers.h"

namespace cq35 {

// With a = max |y_i| of a row: scale = a / 127, q_i = rint(y_i * (127 / a)), half
// to even, so |q_i| is at most 127. A row with a value that is not finite gets the
// scale NaN, one without a magnitude of 127 * 2^-126 (whose scale would lose bits
// in the subnormals) the scale 0, both zeros.
enum class RowSource { kPlain, kNorm, kGated };
constexpr float kLeastAmax = 127.0f * 1.17549435e-38f;

struct RowArgs {
  const void *a, *b;  // rows, and the residual or the up projection
  int64_t a_stride, b_stride;
  void* sum;
  int64_t sum_stride;
  const float* weight;
  float eps;
  int64_t rows;
  int channels;
  int8_t* data;
  int64_t data_stride;
  float* scale;
};

// A 16-byte piece of a row of T.
template <typename T>
struct RowPiece;
template <>
struct RowPiece<uint16_t> {
  static constexpr int kValues = 8;
  static __device__ __forceinline__ void widen(const u32x4& raw, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = lo2f(raw[i]), x[2 * i + 1] = hi2f(raw[i]);
  }
  static __device__ __forceinline__ u32x4 narrow(const float* x) {
    u32x4 raw;
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = (uint32_t)f2bf(x[2 * i]) | (uint32_t)f2bf(x[2 * i + 1]) << 16;
    return raw;
  }
};
template <>
struct RowPiece<float> {
  static constexpr int kValues = 4;
  static __device__ __forceinline__ void widen(const u32x4& raw, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = bitsf(raw[i]);
  }
  static __device__ __forceinline__ u32x4 narrow(const float* x) {
    return u32x4{fbits(x[0]), fbits(x[1]), fbits(x[2]), fbits(x[3])};
  }
};

// Four values, already times 127 / a, rounded half to even: the sum with 1.5 * 2^23 has
// the integer in its low bits.
__device__ __forceinline__ uint32_t pack_int8(const float* v) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = fbits(v[i] + 12582912.0f);
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
  return lo | hi << 16;
}

// g / (1 + e^-g), within 7 half-steps of F32 down to g = -87.3 (e^-g = 2^126), 0 below: e^-g = 2^t (1 + r ln 2) with
// t = -g log2 e rounded and r what its rounding and that of log2 e leave out; 2^t alone was off by up to 1.5 |g|
// half-steps more, and took 1 to 4 % less time (8192 rows of 6144 BF16 48.4 instead of 49.9, of 2048 17.6 and 18.2).
// Gates beyond 128, where e^-g is 0, have 128's exponent, as t of the largest would be infinite and r with it; a
// minimum of their bits as integers leaves negative numbers alone (t is infinite for the largest of those, too, and
// 2^t with it).
__device__ __forceinline__ float gate_of(float g) {
  const float x = bitsf(min((int32_t)fbits(g), 0x43000000)), t = x * -1.44269502f;
  const float r = __builtin_fmaf(x, -1.92596299e-8f, __builtin_fmaf(x, -1.44269502f, -t));
  return g * __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_amdgcn_exp2f(t), __builtin_fmaf(r, 0.693147181f, 1.0f), 1.0f));
}

// kLanes threads a row, kPieces pieces of 16 bytes a thread. Where a wave is a row it goes on to others, the next
// one's pieces asked for under the current one's arithmetic and the norm's weights kept in registers. Sixteen waves
// have 128 registers a thread and 64 values in them: what does not fit beside those is asked for piece by piece, the
// weights behind the sum of squares. Held as in the other widths it went to scratch memory: 4096 rows of 12288
// channels normed with residual 167 us instead of 86 (F32 393, 145), gated F32 132 instead of 93. Gated rows of BF16
// in a wave each are asked to fit in 96 registers, five waves a SIMD: 97 without, and 18.7 us instead of 18.2 for 8192
// rows of 2048.
template <typename T, RowSource kSource, int kLanes, int kPieces>
__global__ __launch_bounds__(kLanes < 256 ? 256 : kLanes, kLanes == 64 && kSource == RowSource::kGated && sizeof(T) == 2 ? 5 : 1) void k_int8_rows(RowArgs a) {
  typedef RowPiece<T> P;
  constexpr int E = P::kValues, kThreads = kLanes < 256 ? 256 : kLanes, kWaves = kLanes / 64, kRows = kThreads / kLanes;
  // registers for a row's pieces and the weights at once, beside its values
  constexpr int kBeside = kPieces * (kSource == RowSource::kPlain ? 4 : 8) + (kSource == RowSource::kNorm ? kPieces * E : 0);
  constexpr bool kHeld = kLanes < 1024 || kBeside <= 64;
  constexpr int kBatch = kHeld ? kPieces : 1;
  __shared__ float sums[kWaves];
  __shared__ uint32_t most[kWaves];
  const int tid = threadIdx.x, lane = tid % kLanes, wave = lane >> 6;
  const bool two = kSource == RowSource::kGated || (kSource == RowSource::kNorm && a.b);
  struct Row {
    u32x4 a[kBatch], b[kSource == RowSource::kPlain ? 1 : kBatch];
  } next;
  auto load = [&](Row& r, int64_t row, int first) {
#pragma unroll
    for (int p = 0; p < kBatch; ++p) {
      const int i = ((first + p) * kLanes + lane) * E;
      if (i >= a.channels) continue;
      r.a[p] = *reinterpret_cast<const u32x4*>((const T*)a.a + row * a.a_stride + i);
      if (kSource != RowSource::kPlain && two) r.b[p] = *reinterpret_cast<const u32x4*>((const T*)a.b + row * a.b_stride + i);
    }
  };
  int64_t row = (int64_t)blockIdx.x * kRows + tid / kLanes;
  if (row >= a.rows) return;  // whole waves; only where a wave is a row
  load(next, row, 0);
  auto load_weights = [&](float* w, int i) {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(a.weight + i + e);
      w[e] = v.x, w[e + 1] = v.y, w[e + 2] = v.z, w[e + 3] = v.w;
    }
  };
  float w[kHeld && kSource == RowSource::kNorm ? kPieces : 1][E];
  if (kHeld && kSource == RowSource::kNorm)
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int i = (p * kLanes + lane) * E;
      if (i < a.channels) load_weights(w[p], i);
    }
  for (;;) {
    Row now = next;
    const int64_t after = row + (int64_t)gridDim.x * kRows;
    if (kLanes == 64 && after < a.rows) load(next, after, 0);
    float y[kPieces][E];
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int i = (p * kLanes + lane) * E;
      if (p > 0 && p % kBatch == 0) load(now, row, p);
#pragma unroll
      for (int e = 0; e < E; ++e) y[p][e] = 0.0f;
      if (i >= a.channels) continue;
      P::widen(now.a[p % kBatch], y[p]);
      if (kSource == RowSource::kNorm && two) {
        float r[E];
        P::widen(now.b[p % kBatch], r);
#pragma unroll
        for (int e = 0; e < E; ++e) y[p][e] += r[e];
        // the sum in the stream's type is what the norm sees
        const u32x4 raw = P::narrow(y[p]);
        *reinterpret_cast<u32x4*>((T*)a.sum + row * a.sum_stride + i) = raw;
        P::widen(raw, y[p]);
      }
      if (kSource == RowSource::kGated) {
        float u[E];
        P::widen(now.b[p % kBatch], u);
#pragma unroll
        for (int e = 0; e < E; ++e) y[p][e] = gate_of(y[p][e]) * u[e];
      }
    }
    if (kSource == RowSource::kNorm) {
      float s = 0.0f;
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
#pragma unroll
        for (int e = 0; e < E; ++e) s = __builtin_fmaf(y[p][e], y[p][e], s);
      s = lanes_sum(s);
      if (kWaves > 1) {
        if ((tid & 63) == 0) sums[wave] = s;
        __syncthreads();
        s = 0.0f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) s += sums[v];
      }
      const float inverse = 1.0f / sqrtf(s / (float)a.channels + a.eps);
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const int i = (p * kLanes + lane) * E;
        if (i >= a.channels) continue;
        if (!kHeld) load_weights(w[0], i);
#pragma unroll
        for (int e = 0; e < E; ++e) y[p][e] = y[p][e] * inverse * w[kHeld ? p : 0][e];
      }
    }
    // magnitudes as integers: infinity and NaN are the largest
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
#pragma unroll
      for (int e = 0; e < E; ++e) m = max(m, fbits(y[p][e]) & 0x7fffffffu);
    m = lanes_max(m);
    if (kWaves > 1) {
      if ((tid & 63) == 0) most[wave] = m;
      __syncthreads();
      m = 0;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) m = max(m, most[v]);
    }
    const float amax = bitsf(m);
    const bool zeros = m >= 0x7f800000u || amax < kLeastAmax;
    // 127 / a in two parts: with the second one y (127 / a) rounds once. Without it the values of a / 2, common among
    // BF16 and 63.5 exactly, were 63 under 14 of the 128 mantissas of a. (2048 channels 9.8 -> 10.0 us for 8192 rows,
    // 6144 29.4 both.)
    const float up = 127.0f / amax, rest = __builtin_fmaf(-up, amax, 127.0f) * up * (1.0f / 127.0f);
    if (lane == 0) a.scale[row] = m >= 0x7f800000u ? bitsf(0x7fc00000u) : zeros ? 0.0f : amax / 127.0f;
    int8_t* to = a.data + row * a.data_stride;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int i = (p * kLanes + lane) * E;
      if (i >= a.channels) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) y[p][e] = zeros ? 0.0f : __builtin_fmaf(y[p][e], up, y[p][e] * rest);
      if (E == 8) *reinterpret_cast<uint2*>(to + i) = make_uint2(pack_int8(y[p]), pack_int8(y[p] + E / 2));
      else *reinterpret_cast<uint32_t*>(to + i) = pack_int8(y[p]);
    }
    if (kLanes != 64 || after >= a.rows) return;
    row = after;
  }
}

}  // namespace cq35
