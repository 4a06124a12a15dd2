// C entry points of the 8-bit rows and products and of the log probabilities:
// argument checks, then the launches on the caller's stream, as the paged-cache
// operators' are.
#pragma once

#include "int8_product.h"
#include "int8_rows.h"
#include "logprobs.h"
#include "operator_call.h"

namespace {

constexpr int64_t kMostRows = 1 << 21;  // times 1024 threads: a launch takes below 2^32
constexpr int64_t kComputeUnits = 256;
constexpr int64_t kRowBlocks = 8 * kComputeUnits;  // where a wave is a row, more rows share a wave
constexpr int64_t kLogprobBlocks = 4 * kComputeUnits;  // more rows take a block each
constexpr int64_t kMostResults = 1ll << 34;  // in tiles of 16 x 16 by 512 threads as well

bool row_type(int32_t dtype) { return dtype == CQ35_BF16 || dtype == CQ35_F32; }

// Rows read or written in 16-byte pieces.
int check_rows(const char* what, const cq35_rows* r, int64_t rows, int64_t channels, bool written) {
  if (!r || !r->data) return fail(CQ35_EINVAL, "%s: null argument", what);
  if (!row_type(r->dtype)) return fail(CQ35_EUNSUPPORTED, "%s: type %d is neither BF16 nor F32", what, r->dtype);
  const int unit = r->dtype == CQ35_BF16 ? 8 : 4;
  if (!aligned16(r->data)) return fail(CQ35_EINVAL, "%s: not at a 16-byte address", what);
  if (r->row_stride < 0 || r->row_stride % unit)
    return fail(CQ35_EINVAL, "%s: rows %lld elements apart, not a multiple of %d", what, (long long)r->row_stride, unit);
  if (written && !distinct({{rows, r->row_stride}}, channels)) return fail(CQ35_EINVAL, "%s: rows overlap", what);
  return CQ35_OK;
}

int check_int8_rows(const char* what, const cq35_int8_rows* r, int64_t rows, int64_t channels, bool written) {
  if (!r || !r->data || !r->scale) return fail(CQ35_EINVAL, "%s: null argument", what);
  if (!aligned16(r->data)) return fail(CQ35_EINVAL, "%s: not at a 16-byte address", what);
  if (r->row_stride < 0 || r->row_stride % 16)
    return fail(CQ35_EINVAL, "%s: rows %lld bytes apart, not a multiple of 16", what, (long long)r->row_stride);
  if (written && !distinct({{rows, r->row_stride}}, channels)) return fail(CQ35_EINVAL, "%s: rows overlap", what);
  return CQ35_OK;
}

int check_row_sizes(const char* what, int64_t rows, int64_t channels) {
  if (rows < 0 || rows > kMostRows) return fail(CQ35_ERANGE, "%s: %lld rows, not up to 2^21", what, (long long)rows);
  if (channels < 16 || channels > kProductMostChannels || channels % 16)
    return fail(CQ35_ERANGE, "%s: %lld channels, not a multiple of 16 up to 65536", what, (long long)channels);
  return CQ35_OK;
}

// A wave a row up to 2048 channels, four up to 8192, sixteen beyond, so that a thread holds 32 values (64): a
// block of four waves takes 2.6 us for 16 rows of 4096 channels, 21.5 for 8192 (100 MB, 4.7 TB/s).
template <typename T, RowSource kSource>
int launch_rows(const char* what, const RowArgs& a, hipStream_t s) {
  constexpr int E = RowPiece<T>::kValues;
  if (a.channels <= 2048)
    return launch_operator(what, k_int8_rows<T, kSource, 64, 32 / E>, dim3((unsigned)std::min<int64_t>((a.rows + 3) / 4, kRowBlocks)), 256, 0, s, a);
  if (a.channels <= 8192) return launch_operator(what, k_int8_rows<T, kSource, 256, 32 / E>, dim3((unsigned)a.rows), 256, 0, s, a);
  return launch_operator(what, k_int8_rows<T, kSource, 1024, 64 / E>, dim3((unsigned)a.rows), 1024, 0, s, a);
}

template <RowSource kSource>
int launch_rows(const char* what, int32_t dtype, const RowArgs& a, hipStream_t s) {
  return dtype == CQ35_BF16 ? launch_rows<uint16_t, kSource>(what, a, s) : launch_rows<float, kSource>(what, a, s);
}

RowArgs row_args(const cq35_rows* x, int64_t rows, int64_t channels, const cq35_int8_rows* out) {
  RowArgs a{};
  a.a = x->data, a.a_stride = x->row_stride, a.rows = rows, a.channels = (int)channels;
  a.data = out->data, a.data_stride = out->row_stride, a.scale = out->scale;
  return a;
}

template <typename T, int BM, int BN>
int launch_tiles(const ProductArgs& a, hipStream_t s) {
  constexpr size_t lds = ProductTile<T, BM, BN>::kLds;
  if (lds > 65536) HIP_TRY(hipFuncSetAttribute((const void*)k_int8_tiles<T, BM, BN>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  const int64_t blocks = ((a.rows + BM - 1) / BM) * ((a.outputs + BN - 1) / BN);
  return launch_operator("int8 linear", k_int8_tiles<T, BM, BN>, dim3((unsigned)blocks), 256, lds, s, a);
}

template <typename T, int MT>
int launch_few(const ProductArgs& a, hipStream_t s) {
  const unsigned blocks = (unsigned)((a.outputs + 15) / 16);
  // more than two blocks a compute unit: the kernel of which four fit
  const bool many = MT > 1 || blocks > 2 * kComputeUnits;
  return launch_operator("int8 linear", many ? k_int8_few<T, MT, 2> : k_int8_few<T, MT, (MT > 1 ? 2 : 4)>, dim3(blocks), 512, 0, s, a);
}

// The kernels and what a block of each takes, in ns: alone on its compute unit, and each further one there, by
// the stages of 64 channels. Fitted to measured times; for 2048 channels to 9216 outputs (us, tiles of 64 x 64,
// 128 x 128, 256 x 128, 256 x 256): 65 rows 10.5, 12.3, 18.4, 28.2; 300 rows 17.3, 13.9, 20.0, 30.7; 512 rows 25.7,
// 21.6, 20.7, 31.1; 4096 rows 163, 105, 93, 103; 8192 rows to 12288 outputs -, 280, 251, 234. Up to 16 rows the
// kernel of few rows takes 4.1 to 4.8 to 2048 outputs (64 x 64: 7.8); one row 6.9 to 12288 (8.1) and 83 to 248320 (90),
// but sixteen 8.6 (8.2) and 140 (111).
// All with operands in the memory-side cache. No kernel divides the channels among blocks, so many channels to few
// outputs leave compute units idle: 33, 64, 128 and 300 rows of 6144 channels to 2048 outputs take 17 to 18, from HBM
// 23 to 25, one row 6.2 and 7.2, 300 rows of 3584 to 1024 11.3; a read of their bytes takes 1 to 3.
struct ProductKernel {
  int rows, outputs;  // of a block
  int most_rows;
  int64_t start, stage, more_start, more_stage;
  int64_t more_row;  // of each row, by the stage
};
constexpr ProductKernel kProductKernels[] = {
    {16, 16, 16, 3000, 40, 500, 18, 2},             {32, 16, 32, 3300, 81, 1000, 62, 0},            {64, 64, INT32_MAX, 3500, 154, 1200, 110, 0},
    {128, 128, INT32_MAX, 4900, 224, 1500, 310, 0}, {256, 128, INT32_MAX, 6700, 360, 1800, 553, 0}, {256, 256, INT32_MAX, 10400, 560, 11000, 867, 0},
};

int product_kernel(int64_t rows, int64_t outputs, int64_t channels) {
  int best = 0;
  int64_t least = INT64_MAX;
  for (int i = 0; i < (int)(sizeof(kProductKernels) / sizeof(kProductKernels[0])); ++i) {
    const ProductKernel& k = kProductKernels[i];
    if (rows > k.most_rows) continue;
    const int64_t blocks = ((rows + k.rows - 1) / k.rows) * ((outputs + k.outputs - 1) / k.outputs);
    const int64_t stages = (channels + 63) / 64, more = (blocks + kComputeUnits - 1) / kComputeUnits - 1;
    const int64_t time = k.start + stages * k.stage + more * (k.more_start + stages * (k.more_stage + rows * k.more_row));
    if (time < least) best = i, least = time;
  }
  return best;
}

template <typename T>
int launch_product(const ProductArgs& a, hipStream_t s) {
  switch (product_kernel(a.rows, a.outputs, a.channels)) {
    case 0: return launch_few<T, 1>(a, s);
    case 1: return launch_few<T, 2>(a, s);
    case 2: return launch_tiles<T, 64, 64>(a, s);
    case 3: return launch_tiles<T, 128, 128>(a, s);
    case 4: return launch_tiles<T, 256, 128>(a, s);
    default: return launch_tiles<T, 256, 256>(a, s);
  }
}

}  // namespace

extern "C" int cq35_quantize_rows(const cq35_rows* x, int64_t rows, int64_t channels, const cq35_int8_rows* out,
                                  void* stream) {
  int rc = check_row_sizes("quantize rows", rows, channels);
  if (rc || rows == 0) return rc;
  rc = check_rows("quantize rows: input", x, rows, channels, false);
  if (!rc) rc = check_int8_rows("quantize rows: output", out, rows, channels, true);
  if (rc) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  OperatorDevice on;
  rc = on.enter({x->data, out->data, out->scale}, s);
  if (rc) return rc;
  return launch_rows<RowSource::kPlain>("quantize rows", x->dtype, row_args(x, rows, channels, out), s);
}

extern "C" int cq35_norm_quantize(const cq35_rows* x, const cq35_rows* residual, const float* weight, float eps,
                                  int64_t rows, int64_t channels, const cq35_rows* summed, const cq35_int8_rows* out,
                                  void* stream) {
  int rc = check_row_sizes("norm quantize", rows, channels);
  if (rc) return rc;
  if (!(eps >= 0.0f)) return fail(CQ35_EINVAL, "norm quantize: eps %g", (double)eps);
  if (rows == 0) return CQ35_OK;
  if (!weight) return fail(CQ35_EINVAL, "norm quantize: null argument");
  if (!aligned16(weight)) return fail(CQ35_EINVAL, "norm quantize: weights not at a 16-byte address");
  rc = check_rows("norm quantize: input", x, rows, channels, false);
  if (!rc && residual) rc = check_rows("norm quantize: residual", residual, rows, channels, false);
  if (!rc && residual) rc = check_rows("norm quantize: sum", summed, rows, channels, true);
  if (!rc) rc = check_int8_rows("norm quantize: output", out, rows, channels, true);
  if (rc) return rc;
  if (residual && (residual->dtype != x->dtype || summed->dtype != x->dtype))
    return fail(CQ35_EINVAL, "norm quantize: input, residual and sum of types %d, %d and %d", x->dtype, residual->dtype, summed->dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  OperatorDevice on;
  rc = on.enter({x->data, weight, residual ? residual->data : nullptr, residual ? summed->data : nullptr, out->data, out->scale}, s);
  if (rc) return rc;
  RowArgs a = row_args(x, rows, channels, out);
  a.weight = weight, a.eps = eps;
  if (residual) a.b = residual->data, a.b_stride = residual->row_stride, a.sum = summed->data, a.sum_stride = summed->row_stride;
  return launch_rows<RowSource::kNorm>("norm quantize", x->dtype, a, s);
}

extern "C" int cq35_gated_quantize(const cq35_rows* gate, const cq35_rows* up, int64_t rows, int64_t channels,
                                   const cq35_int8_rows* out, void* stream) {
  int rc = check_row_sizes("gated quantize", rows, channels);
  if (rc || rows == 0) return rc;
  rc = check_rows("gated quantize: gate", gate, rows, channels, false);
  if (!rc) rc = check_rows("gated quantize: up", up, rows, channels, false);
  if (!rc) rc = check_int8_rows("gated quantize: output", out, rows, channels, true);
  if (rc) return rc;
  if (gate->dtype != up->dtype) return fail(CQ35_EINVAL, "gated quantize: gate and up of types %d and %d", gate->dtype, up->dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  OperatorDevice on;
  rc = on.enter({gate->data, up->data, out->data, out->scale}, s);
  if (rc) return rc;
  RowArgs a = row_args(gate, rows, channels, out);
  a.b = up->data, a.b_stride = up->row_stride;
  return launch_rows<RowSource::kGated>("gated quantize", gate->dtype, a, s);
}

extern "C" int cq35_int8_linear(const cq35_int8_rows* x, const cq35_int8_rows* w, int64_t rows, int64_t outputs,
                                int64_t channels, const cq35_rows* out, void* stream) {
  int rc = check_row_sizes("int8 linear", rows, channels);
  if (rc) return rc;
  if (outputs < 1 || outputs > kMostRows) return fail(CQ35_ERANGE, "int8 linear: %lld outputs, not 1 to 2^21", (long long)outputs);
  if (rows * outputs > kMostResults)
    return fail(CQ35_ERANGE, "int8 linear: too many results for one call: %lld x %lld", (long long)rows, (long long)outputs);
  if (rows == 0) return CQ35_OK;
  rc = check_int8_rows("int8 linear: input", x, rows, channels, false);
  if (!rc) rc = check_int8_rows("int8 linear: weights", w, outputs, channels, false);
  if (rc) return rc;
  if (!out || !out->data) return fail(CQ35_EINVAL, "int8 linear: output: null argument");
  if (!row_type(out->dtype)) return fail(CQ35_EUNSUPPORTED, "int8 linear: output: type %d is neither BF16 nor F32", out->dtype);
  if ((uintptr_t)out->data % (out->dtype == CQ35_BF16 ? 2 : 4)) return fail(CQ35_EINVAL, "int8 linear: output: misaligned");
  if (out->row_stride < 0 || !distinct({{rows, out->row_stride}}, outputs)) return fail(CQ35_EINVAL, "int8 linear: output: rows overlap");
  hipStream_t s = static_cast<hipStream_t>(stream);
  OperatorDevice on;
  rc = on.enter({x->data, x->scale, w->data, w->scale, out->data}, s);
  if (rc) return rc;
  const ProductArgs a{x->data, w->data, x->row_stride, w->row_stride, x->scale, w->scale, rows, outputs, (int)channels,
                      out->data, out->row_stride};
  return out->dtype == CQ35_BF16 ? launch_product<uint16_t>(a, s) : launch_product<float>(a, s);
}

namespace {

int check_logprob_sizes(const char* what, int64_t rows, int64_t vocab, int64_t given, int32_t top) {
  if (rows < 0 || rows > kMostRows || vocab < 1 || vocab > 1 << 30)
    return fail(CQ35_ERANGE, "%s: %lld rows of %lld logits", what, (long long)rows, (long long)vocab);
  if (given < 0 || given > kLogprobsMostGiven)
    return fail(CQ35_ERANGE, "%s: %lld given tokens a row, not up to %d", what, (long long)given, kLogprobsMostGiven);
  if (top < 0 || top > kLogprobsMostTop || top > vocab)
    return fail(CQ35_ERANGE, "%s: %d alternatives, not up to %d", what, top, (int)std::min<int64_t>(vocab, kLogprobsMostTop));
  return CQ35_OK;
}

// Blocks of a row, and the bytes of workspace they need.
struct LogprobPlan {
  int splits;
  int64_t keys_at, bytes;
};
LogprobPlan plan_logprobs(int64_t rows, int64_t vocab, int32_t top) {
  const int64_t tiles = (vocab + LogitTile<uint16_t>::kLogits - 1) / LogitTile<uint16_t>::kLogits;  // of BF16, half as many as of F32
  const int64_t wanted = std::max<int64_t>(1, kLogprobBlocks / std::max<int64_t>(rows, 1));
  LogprobPlan p{(int)std::min<int64_t>({tiles, wanted, (int64_t)kLogprobMostSplits}), 0, 0};
  if (p.splits > 1) p.keys_at = 16 * rows * p.splits, p.bytes = p.keys_at + 8 * rows * p.splits * top;
  return p;
}

template <typename T>
int launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  const int rc = launch_operator("token logprobs", a.top ? k_logprobs<T, true> : k_logprobs<T, false>, dim3((unsigned)(a.rows * a.splits)),
                                 kLogprobThreads, 0, s, a);
  if (rc || a.splits == 1) return rc;
  return launch_operator("token logprobs", k_logprobs_join<T>, dim3((unsigned)a.rows), kLogprobThreads, 0, s, a);
}

}  // namespace

extern "C" int cq35_token_logprobs_workspace(int64_t rows, int64_t vocab, int64_t given, int32_t top, int64_t* bytes) {
  if (!bytes) return fail(CQ35_EINVAL, "token logprobs workspace: null argument");
  const int rc = check_logprob_sizes("token logprobs workspace", rows, vocab, given, top);
  if (!rc) *bytes = rows ? plan_logprobs(rows, vocab, top).bytes : 0;
  return rc;
}

extern "C" int cq35_token_logprobs(const cq35_rows* logits, int64_t rows, int64_t vocab, const int64_t* tokens,
                                   int64_t given, int32_t top, float* logprobs, float* entropy, int64_t* top_tokens,
                                   float* top_logprobs, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_logprob_sizes("token logprobs", rows, vocab, given, top);
  if (rc || rows == 0) return rc;
  if (!logits || !logits->data || !entropy || (given > 0 && (!tokens || !logprobs)) || (top > 0 && (!top_tokens || !top_logprobs)))
    return fail(CQ35_EINVAL, "token logprobs: null argument");
  if (!row_type(logits->dtype)) return fail(CQ35_EUNSUPPORTED, "token logprobs: type %d is neither BF16 nor F32", logits->dtype);
  if ((uintptr_t)logits->data % (logits->dtype == CQ35_BF16 ? 2 : 4) || logits->row_stride < 0)
    return fail(CQ35_EINVAL, "token logprobs: logits misaligned, or rows %lld apart", (long long)logits->row_stride);
  const LogprobPlan p = plan_logprobs(rows, vocab, top);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || !aligned16(workspace)))
    return fail(CQ35_EINVAL, "token logprobs: %lld bytes of workspace at a 16-byte address needed, %lld given", (long long)p.bytes,
                (long long)(workspace ? workspace_bytes : 0));
  hipStream_t s = static_cast<hipStream_t>(stream);
  OperatorDevice on;
  rc = on.enter({logits->data, entropy, given ? tokens : nullptr, given ? logprobs : nullptr, top ? top_tokens : nullptr,
                 top ? top_logprobs : nullptr, p.bytes ? workspace : nullptr}, s);
  if (rc) return rc;
  const LogprobArgs a{logits->data, logits->row_stride, rows, (int)vocab, tokens, (int)given, top, logprobs, entropy, top_tokens,
                      top_logprobs, p.splits, (float*)workspace, (uint64_t*)((char*)workspace + p.keys_at)};
  return logits->dtype == CQ35_BF16 ? launch_logprobs<uint16_t>(a, s) : launch_logprobs<float>(a, s);
}
