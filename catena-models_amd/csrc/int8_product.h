// Product of 8-bit rows: out[m][n] = (sum_k x[m][k] w[n][k]) sx[m] sw[n], the sums
// exact in 32-bit integers (channels <= 2^16, so they stay below 2^30), the two
// products and the rounding of the sum to F32 one rounding each, the result rounded once
// more where it is BF16.
//
// Few rows are bound by the weights' bytes and by latency: one row of 2048 channels to 12288 outputs 6.9 us with the
// weights in the 256 MB memory-side cache, 8.4 from HBM (3.0 TB/s), to 248320 outputs 81 (6.3), to 2048 4.1. Large
// products are bound by the card's power: 8192 rows of 8192 channels to 8192 outputs 490 us, 2.2 POP/s, the matrix
// cores busy 0.61 of the cycles at 1.65 to 1.8 GHz; with nothing fetched the same loop keeps them busy 0.76 at 2.2
// GHz. Those of fewer channels add a tile's start and end, 10 us of 256 x 256 results: 8192 rows of 2048 to 12288
// outputs 245 us, 1.68 POP/s. In between LDS is the bound: the waves' reads and the requests' writes share its port,
// 64 channels of a 128 x 128 tile take about 550 cycles there and 256 on the matrix cores.
#pragma once

#include "layers.h"
#include "paged_attention.h"

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

__device__ __align__(16) uint32_t product_zeros[4];

__device__ __forceinline__ void store_four(float a, float b, float c, float d, uint16_t* to) {
  *reinterpret_cast<uint2*>(to) = make_uint2((uint32_t)f2bf(a) | (uint32_t)f2bf(b) << 16, (uint32_t)f2bf(c) | (uint32_t)f2bf(d) << 16);
}
__device__ __forceinline__ void store_one(float v, uint16_t* to) { *to = f2bf(v); }
__device__ __forceinline__ void store_one(float v, float* to) { *to = v; }
__device__ __forceinline__ void store_four(float a, float b, float c, float d, float* to) {
  *reinterpret_cast<float4*>(to) = make_float4(a, b, c, d);
}

// Block = BM rows x BN outputs, four waves of half by half. Channels go through LDS 64 a stage by
// DMA, kStages stages, one barrier a stage; a stage holds BM + BN rows of 64 bytes whose
// 16-byte pieces are swapped so that sixteen neighbouring rows' same piece lie in different ones of the 64
// banks (swapped by the next lower bit of the row half of the reads' cycles were conflicts). Weights are the
// first operand of the matrix instruction, so that a lane's results are four neighbouring outputs of one row.
//
// Measured and not kept (8192 rows of 2048 channels to 12288 outputs unless said otherwise): products of 16 x 16
// with whole stages in registers, spilled at 256 x 256 (397 us) and 10 % faster at 64 x 64; requests all behind the
// barrier instead of spread (259 against 248); two groups of waves with half the channels each, joined in LDS (300
// rows to 9216 17.1 us against 14.6); rings of 8 or 16 stages (no change); a block that goes on to further tiles,
// their first stages requested under the stores (250 to 274 against 245: the compiler copies the sums); stores past
// the caches (238 against 232); tiles of 64 x 128
// (4096 rows: 182 us against 138 of 128 x 128); the waves side by side along the outputs, 32 each, whose weights go
// from memory straight to registers eight stages ahead and only rows through LDS (300 rows to 9216 17.6 against 15.2,
// 8192 rows 337 to 364: 16 bytes from each of 32 rows are 64 requests to the caches, four times those of 1 KB by DMA).
template <typename T, int BM, int BN>
struct ProductTile {
  static constexpr int kStage = (BM + BN) * 64, kStages = BM * BN == 256 * 128 ? 3 : 4;  // two blocks of 256 x 128 a CU
  static constexpr int TM = BM / 64, TN = BN / 64;     // tiles of 32 of a wave
  static constexpr int kLoads = (BM + BN) / 16 / 4;    // requests of a wave and stage
  static constexpr int kEarly = kLoads / 2;            // made with the second half of the products of the stage before
  static constexpr int kSlabRow = BN / 2 * sizeof(T) + 16;  // bytes of a row of results in LDS
  static constexpr int kSlabs = 4 * 32 * kSlabRow;
  static constexpr int kScales = kStages * kStage > kSlabs ? kStages * kStage : kSlabs;  // of outputs and rows, behind the rest
  static constexpr size_t kLds = kScales + (BM + BN) * sizeof(float);
};

// Blocks go round the eight XCDs; each XCD takes a run of tiles, ordered in bands of kBand tiles down so
// that the 32 at work on it at a time share rows and weights in its L2.
struct TilePlace {
  uint32_t down, across;
};
constexpr uint32_t kBand = 8;
__device__ __forceinline__ TilePlace tile_place(uint32_t block, uint32_t blocks, uint32_t down) {
  const uint32_t xcd = block & 7, per = blocks >> 3, more = blocks & 7;
  const uint32_t at = xcd * per + min(xcd, more) + (block >> 3);
  const uint32_t across = blocks / down, band = at / (kBand * across), first = band * kBand;
  const uint32_t height = min(kBand, down - first), inside = at - first * across;
  return {first + inside % height, inside / height};
}

__device__ __forceinline__ int piece_swap(int row) { return row >> 2 & 3; }

template <typename T, int BM, int BN>
__global__ __launch_bounds__(256, BM * BN > 256 * 128 ? 1 : 2) void k_int8_tiles(ProductArgs a) {
  typedef ProductTile<T, BM, BN> P;
  extern __shared__ __align__(1024) uint8_t product_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const TilePlace place = tile_place(blockIdx.x, gridDim.x, (uint32_t)((a.rows + BM - 1) / BM));
  const int64_t m0 = (int64_t)place.down * BM, n0 = (int64_t)place.across * BN;
  const uint32_t lds = lds_address(product_lds);
  // what the lane requests: a piece of 16 rows
  const int8_t* from[P::kLoads];
  const int from_row = lane >> 2, piece = 16 * ((lane & 3) ^ piece_swap(from_row));
#pragma unroll
  for (int u = 0; u < P::kLoads; ++u) {
    const int q = wave * P::kLoads + u;
    from[u] = piece + (q < BM / 16 ? a.x + min(m0 + q * 16 + from_row, a.rows - 1) * a.x_stride
                                   : a.w + min(n0 + (q - BM / 16) * 16 + from_row, a.outputs - 1) * a.w_stride);
  }
  float* scales = reinterpret_cast<float*>(product_lds + P::kScales);
  // the thread's share of the scales, under way with the first stages
  float sw = 0.0f, sx = 0.0f;
  if (threadIdx.x < BN) sw = a.sw[min(n0 + threadIdx.x, a.outputs - 1)];
  if (threadIdx.x < BM) sx = a.sx[min(m0 + threadIdx.x, a.rows - 1)];
  const int stages = (a.channels + 63) / 64;
  // Zeros behind the last channel, and for stages behind the last: the loop has one body and no other way
  // through it, as the compiler would copy the sums where ways meet.
  auto request = [&](int i, int u) {
    const uint32_t to = lds + (uint32_t)(i % P::kStages) * P::kStage + (wave * P::kLoads + u) * 1024;
    request_lds(to, 64 * i + piece >= a.channels ? reinterpret_cast<const int8_t*>(product_zeros) : from[u]);
    from[u] += 64;
  };
  i32x16 acc[P::TM][P::TN] = {};
  const int wm = (wave & 1) * BM / 2, wn = (wave >> 1) * BN / 2;
  // the lane's pieces of both halves of a stage
  uint32_t x_at[2], w_at[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint32_t at = 64 * c + 16 * ((2 * s + h) ^ piece_swap(c));
    x_at[s] = at + 64 * wm, w_at[s] = at + 64 * (BM + wn);
  }
  i32x4 f[2][P::TM + P::TN];
  auto read = [&](int i, int s, int t) {
    const uint8_t* stage = product_lds + (i % P::kStages) * P::kStage;
    f[s][t] = *reinterpret_cast<const i32x4*>(t < P::TM ? stage + x_at[s] + 2048 * t : stage + w_at[s] + 2048 * (t - P::TM));
  };
  // The products of half s of a stage, and between them the reads of the next half and half of a stage's
  // requests: a matrix instruction takes 32 cycles, in which others issue. The requests lie apart, as the four
  // waves' go through one unit at 16 cycles each.
  auto multiply = [&](int s, auto next, auto requests, auto load) {
    constexpr int kProducts = P::TM * P::TN, kReads = P::TM + P::TN, kRequests = decltype(requests)::value;
#pragma unroll
    for (int j = 0; j < kProducts; ++j) {
      const int m = j % P::TM, n = j / P::TM;
      acc[m][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[s][P::TM + n], f[s][m], acc[m][n], 0, 0, 0);
#pragma unroll
      for (int t = 0; t < kReads; ++t)
        if ((kReads > kProducts ? t * kProducts / kReads : t) == j) next(t);
#pragma unroll
      for (int u = 0; u < kRequests; ++u)
        if (((u + 1) * kProducts + kRequests - 1) / kRequests - 1 == j) load(u);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // The stage behind the current one is in LDS for every wave, the current one done with.
  auto enter = [&] {
    arrived_but<(P::kStages - 2) * P::kLoads>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll 1
  for (int i = 0; i < P::kStages - 1; ++i)
#pragma unroll
    for (int u = 0; u < P::kLoads; ++u) request(i, u);
  enter();
#pragma unroll
  for (int u = 0; u < P::kEarly; ++u) request(P::kStages - 1, u);
#pragma unroll
  for (int t = 0; t < P::TM + P::TN; ++t) read(0, 0, t);
#pragma unroll 1
  for (int i = 0; i < stages; ++i) {
    multiply(0, [&](int t) { read(i, 1, t); }, std::integral_constant<int, P::kLoads - P::kEarly>{},
             [&](int u) { request(i + P::kStages - 1, P::kEarly + u); });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage's reads are in registers
    enter();
    multiply(1, [&](int t) { read(i + 1, 0, t); }, std::integral_constant<int, P::kEarly>{},
             [&](int u) { request(i + P::kStages, u); });
  }
  arrived_but<0>();
  if (threadIdx.x < BN) scales[threadIdx.x] = sw;
  if (threadIdx.x < BM) scales[BN + threadIdx.x] = sx;
  __syncthreads();
  // Results by rows: 32 rows of the wave's part at a time through LDS, so that a store is of whole lines.
  uint8_t* slab = product_lds + wave * 32 * P::kSlabRow;
  constexpr int V = 16 / sizeof(T), kLanes = BN / 2 / V, kRows = 64 / kLanes;  // lanes of a row of results, rows of a store
  const bool whole = n0 + BN <= a.outputs && ((uintptr_t)a.out | (uintptr_t)(a.out_stride * sizeof(T))) % 16 == 0;
  const int lr = lane / kLanes, at = lane % kLanes * V;
  T* out = (T*)a.out + (m0 + wm + lr) * a.out_stride + n0 + wn + at;
  const T* in = reinterpret_cast<const T*>(slab + lr * P::kSlabRow) + at;
#pragma unroll
  for (int t = 0; t < P::TM; ++t) {
    const float row = scales[BN + wm + 32 * t + c];
#pragma unroll
    for (int n = 0; n < P::TN; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 s = *reinterpret_cast<const float4*>(scales + wn + 32 * n + 8 * g + 4 * h);
        const i32x16& v = acc[t][n];
        store_four((float)v[4 * g] * row * s.x, (float)v[4 * g + 1] * row * s.y, (float)v[4 * g + 2] * row * s.z,
                   (float)v[4 * g + 3] * row * s.w, reinterpret_cast<T*>(slab + c * P::kSlabRow) + 32 * n + 8 * g + 4 * h);
      }
    __builtin_amdgcn_wave_barrier();
    if (whole) {
      u32x4 v[32 / kRows];
#pragma unroll
      for (int r = 0; r < 32 / kRows; ++r) v[r] = *reinterpret_cast<const u32x4*>(in + r * kRows * (P::kSlabRow / sizeof(T)));
#pragma unroll
      for (int r = 0; r < 32 / kRows; ++r)
        if (m0 + wm + 32 * t + r * kRows + lr < a.rows) *reinterpret_cast<u32x4*>(out + (32 * t + r * kRows) * a.out_stride) = v[r];
    } else {
#pragma unroll 1
      for (int r = 0; r < 32; r += kRows)
        for (int e = 0; e < V; ++e)
          if (m0 + wm + 32 * t + r + lr < a.rows && n0 + wn + at + e < a.outputs)
            out[(32 * t + r) * a.out_stride + e] = in[r * (P::kSlabRow / sizeof(T)) + e];
    }
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Few rows: the weights' bytes are the time, so they go from memory straight to registers. Block = 16 MT
// rows x 16 outputs, the channels dealt to its eight waves 128 at a time (a line of memory); a wave keeps
// kAhead runs of 128 under way. The waves' sums meet in LDS by integer additions, whose order changes nothing.
// Two runs leave room for four blocks on a compute unit instead of two, four are longer under way where there are
// fewer blocks: one row of 2048 channels to 12288 outputs 6.9 us with two, 7.8 with four, of 6144 channels to 2048
// outputs 6.5 and 6.3, of 4096 to 4096 6.65 and 6.25. Blocks of four waves: 7.0, 7.6, 7.1 at best; of sixteen as of
// eight (16384 channels to 1024 outputs 11.5 both: a compute unit takes in its 16 rows of weights no faster).
template <typename T, int MT, int kAhead>
__global__ __launch_bounds__(512) void k_int8_few(ProductArgs a) {
  constexpr int kWaves = 8, kFourth = 64 * MT + 16;
  // [e][row][h] of output 4 h + e, so that a wave's 64 sums lie in different banks
  __shared__ int32_t sums[4 * kFourth];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, h = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int8_t* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) x[m] = a.x + min((int64_t)16 * m + c, a.rows - 1) * a.x_stride + 16 * h;
  const int8_t* w = a.w + min(n0 + c, a.outputs - 1) * a.w_stride + 16 * h;
  struct Run {
    i32x4 x[2][MT], w[2];
  } run[kAhead];
  auto load = [&](Run& r, int k) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = k + 64 * s;
      const bool in = at + 16 * h < a.channels;
      r.w[s] = in ? *reinterpret_cast<const i32x4*>(w + at) : i32x4{};
#pragma unroll
      for (int m = 0; m < MT; ++m) r.x[s][m] = in ? *reinterpret_cast<const i32x4*>(x[m] + at) : i32x4{};
    }
  };
  i32x4 acc[MT] = {};
#pragma unroll
  for (int d = 0; d < kAhead; ++d) load(run[d], 128 * (wave + kWaves * d));
  for (int i = threadIdx.x; i < 4 * kFourth; i += 512) sums[i] = 0;
  for (int k = 128 * wave; k < a.channels; k += 128 * kWaves * kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(run[d].w[s], run[d].x[s][m], acc[m], 0, 0, 0);
      load(run[d], k + 128 * kWaves * (kAhead + d));
    }
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) atomicAdd(&sums[e * kFourth + 4 * (16 * m + c) + h], acc[m][e]);
  __syncthreads();
  for (int i = threadIdx.x; i < 256 * MT; i += 512) {
    const int64_t m = i / 16, n = n0 + i % 16;
    const int32_t sum = sums[i % 4 * kFourth + 4 * m + i % 16 / 4];
    if (m < a.rows && n < a.outputs) store_one((float)sum * a.sx[m] * a.sw[n], (T*)a.out + m * a.out_stride + n);
  }
}

}  // namespace cq35
