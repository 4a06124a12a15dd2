// C entry points of the paged-cache operators: argument checks, then the
// launches on the caller's stream. Nothing is allocated, cleared through a
// runtime call or waited for, so every call may be captured into a graph.
#pragma once

#include "paged.h"
#include "paged_attention.h"

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// The device that every one of the pointers lies on; the calling thread's
// device for the length of an operator and back again after it.
class OperatorDevice {
 public:
  ~OperatorDevice() {
    if (before_ >= 0) hipSetDevice(before_);
  }
  int enter(std::initializer_list<const void*> pointers, hipStream_t stream) {
    int device = -1;
    for (const void* p : pointers) {
      if (!p) continue;
      hipPointerAttribute_t at;
      if (hipPointerGetAttributes(&at, p) != hipSuccess ||
          (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)) {
        hipGetLastError();
        return fail(CQ35_EINVAL, "%p is not device memory", p);
      }
      if (device >= 0 && at.device != device)
        return fail(CQ35_EINVAL, "operands lie on devices %d and %d", device, at.device);
      device = at.device;
    }
    hipDevice_t of = 0;
    if (stream) {
      HIP_TRY(hipStreamGetDevice(stream, &of));
      if ((int)of != device) return fail(CQ35_EINVAL, "the stream is device %d's, the operands device %d's", (int)of, device);
    }
    int now = -1;
    HIP_TRY(hipGetDevice(&now));
    if (now != device) {
      HIP_TRY(hipSetDevice(device));
      before_ = now;
    }
    return CQ35_OK;
  }

 private:
  int before_ = -1;
};

template <typename Args>
int launch_operator(const char* what, void (*kernel)(Args), dim3 grid, int threads, size_t lds, hipStream_t stream,
                    Args args) {
  void* list[] = {&args};
  const hipError_t e = hipLaunchKernel((const void*)kernel, grid, dim3((unsigned)threads), list, lds, stream);
  if (e != hipSuccess) {
    hipGetLastError();
    return fail(CQ35_EDEVICE, "%s: %s", what, hipGetErrorString(e));
  }
  return CQ35_OK;
}

// log2 of a page size this build takes, or -1.
int page_shift(int32_t rows) {
  for (int s = 4; s <= 16; ++s)
    if (rows == 1 << s) return s;
  return -1;
}

// Whether dimensions of the given lengths and strides (elements) address
// every element once: in some order each stride covers what lies inside it.
struct Dim {
  int64_t length, stride;
};
template <int N>
bool distinct(const Dim (&dims)[N], int64_t inner) {
  Dim by[N];
  int n = 0;
  for (const Dim& d : dims)
    if (d.length > 1) {
      int i = n++;
      for (; i > 0 && by[i - 1].stride > d.stride; --i) by[i] = by[i - 1];
      by[i] = d;
    }
  int64_t extent = inner;
  for (int i = 0; i < n; ++i) {
    if (by[i].stride < extent || by[i].stride > INT64_MAX / 4 / by[i].length) return false;
    extent += (by[i].length - 1) * by[i].stride;
  }
  return true;
}

int check_heads(const char* what, const cq35_heads* h, int64_t rows, int64_t heads, int head_dim, bool written) {
  if (!h || !h->data) return fail(CQ35_EINVAL, "%s: null argument", what);
  if (!aligned16(h->data)) return fail(CQ35_EINVAL, "%s: not at a 16-byte address", what);
  if (h->row_stride < 0 || h->head_stride < 0 || h->row_stride % 8 || h->head_stride % 8)
    return fail(CQ35_EINVAL, "%s: strides %lld, %lld are not multiples of 8 elements", what, (long long)h->row_stride,
                (long long)h->head_stride);
  if (written && !distinct({{rows, h->row_stride}, {heads, h->head_stride}}, head_dim))
    return fail(CQ35_EINVAL, "%s: rows or heads overlap", what);
  return CQ35_OK;
}

int check_cache(const cq35_paged_cache* c) {
  if (!c || !c->keys || !c->values) return fail(CQ35_EINVAL, "paged cache: null argument");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(CQ35_EUNSUPPORTED, "paged cache: head_dim %d is not 64, 128 or 256", c->head_dim);
  if (c->kv_heads < 1 || c->kv_heads > 1024) return fail(CQ35_EINVAL, "paged cache: %d heads", c->kv_heads);
  if (page_shift(c->page_size) < 0)
    return fail(CQ35_EUNSUPPORTED, "paged cache: page size %d is not a power of two from 16 to 65536", c->page_size);
  if (c->pages < 1 || c->pages > INT32_MAX / c->page_size)
    return fail(CQ35_ERANGE, "paged cache: %lld pages of %d rows", (long long)c->pages, c->page_size);
  if (!aligned16(c->keys) || !aligned16(c->values)) return fail(CQ35_EINVAL, "paged cache: not at a 16-byte address");
  if (c->page_stride < 0 || c->row_stride < 0 || c->head_stride < 0 || c->page_stride % 8 || c->row_stride % 8 ||
      c->head_stride % 8)
    return fail(CQ35_EINVAL, "paged cache: strides %lld, %lld, %lld are not multiples of 8 elements",
                (long long)c->page_stride, (long long)c->row_stride, (long long)c->head_stride);
  if (c->row_stride > 1 << 26) return fail(CQ35_EUNSUPPORTED, "paged cache: rows %lld elements apart", (long long)c->row_stride);
  if (!distinct({{c->pages, c->page_stride}, {c->page_size, c->row_stride}, {c->kv_heads, c->head_stride}}, c->head_dim))
    return fail(CQ35_EINVAL, "paged cache: pages, rows or heads overlap");
  return CQ35_OK;
}

int check_q_heads(const cq35_paged_cache* c, int32_t q_heads) {
  if (q_heads < 1 || q_heads % c->kv_heads || q_heads > 4096)
    return fail(CQ35_EINVAL, "%d query heads over %d key/value heads", q_heads, c->kv_heads);
  return CQ35_OK;
}

}  // namespace

extern "C" int cq35_page_plan(int32_t* table, int64_t table_stride, int64_t requests, int64_t width,
                              const int32_t* cached, const int32_t* lengths, int32_t* free_pages, int64_t pages,
                              const int32_t* free_count, int32_t page_size, int64_t rows, int32_t* row_start,
                              int32_t* positions, int32_t* slots, int32_t* free_left, int32_t* status, void* stream) {
  if (!table || !cached || !lengths || !free_pages || !free_count || !row_start || !free_left || !status ||
      (rows > 0 && (!positions || !slots)))
    return fail(CQ35_EINVAL, "page plan: null argument");
  const int shift = page_shift(page_size);
  if (shift < 0)
    return fail(CQ35_EUNSUPPORTED, "page plan: page size %d is not a power of two from 16 to 65536", page_size);
  if (requests < 1 || requests > kPlanMostRequests)
    return fail(CQ35_ERANGE, "page plan: %lld requests, not 1..%d", (long long)requests, kPlanMostRequests);
  if (pages < 1 || pages > INT32_MAX / page_size || width < 1 || width > INT32_MAX / page_size || rows < 0 ||
      rows > INT32_MAX)
    return fail(CQ35_ERANGE, "page plan: %lld pages, tables of %lld, %lld rows", (long long)pages, (long long)width,
                (long long)rows);
  if (table_stride < width) return fail(CQ35_EINVAL, "page plan: table rows overlap");
  if (free_left == free_count) return fail(CQ35_EINVAL, "page plan: the count left may not take the place of the count before");
  hipStream_t s = static_cast<hipStream_t>(stream);
  OperatorDevice on;
  int rc = on.enter({table, cached, lengths, free_pages, free_count, row_start, rows ? positions : nullptr,
                     rows ? slots : nullptr, free_left, status}, s);
  if (rc) return rc;
  const PlanArgs a{table, table_stride, (int)requests, width, cached, lengths, free_pages, pages, free_count, shift,
                   rows, row_start, positions, slots, free_left, status};
  const size_t lds = plan_lds_bytes((int)requests);
  if (lds > 65536) HIP_TRY(hipFuncSetAttribute((const void*)k_page_plan, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  const int64_t blocks = std::min<int64_t>(std::max<int64_t>((rows + kPlanThreads - 1) / kPlanThreads, 1), 256);
  return launch_operator("page plan", k_page_plan, dim3((unsigned)blocks), kPlanThreads, lds, s, a);
}

extern "C" int cq35_paged_prepare(const cq35_paged_cache* cache, const cq35_heads* q, const cq35_heads* k,
                                  const cq35_heads* v, int64_t rows, int32_t q_heads, const float* q_weight,
                                  const float* k_weight, float eps, const float* inv_freq, int32_t rope_dim,
                                  const int32_t* positions, int64_t position_stride, int32_t axes,
                                  const uint8_t* pair_axis, const int32_t* slots, const cq35_heads* q_out,
                                  void* stream) {
  int rc = check_cache(cache);
  if (!rc) rc = check_q_heads(cache, q_heads);
  if (rc) return rc;
  if (rows < 0 || rows > 1 << 26) return fail(CQ35_ERANGE, "paged prepare: %lld rows, not up to 2^26", (long long)rows);
  if (rope_dim < 16 || rope_dim > cache->head_dim || rope_dim % 16)
    return fail(CQ35_EINVAL, "paged prepare: rotary width %d of heads of %d is not a multiple of 16", rope_dim,
                cache->head_dim);
  if (axes < 1 || axes > 4) return fail(CQ35_EINVAL, "paged prepare: %d position axes, not 1..4", axes);
  if (axes > 1 && !pair_axis) return fail(CQ35_EINVAL, "paged prepare: %d position axes without each pair's axis", axes);
  if (pair_axis)
    for (int i = 0; i < rope_dim / 2; ++i)
      if (pair_axis[i] >= axes) return fail(CQ35_EINVAL, "paged prepare: pair %d on axis %d of %d", i, pair_axis[i], axes);
  if (!(eps >= 0.0f)) return fail(CQ35_EINVAL, "paged prepare: eps %g", (double)eps);
  if (rows == 0) return CQ35_OK;
  if (!q_weight || !k_weight || !inv_freq || !positions || !slots) return fail(CQ35_EINVAL, "paged prepare: null argument");
  if (!aligned16(q_weight) || !aligned16(k_weight)) return fail(CQ35_EINVAL, "paged prepare: norm weights not at a 16-byte address");
  if (axes > 1 && position_stride != 0 && position_stride < rows) return fail(CQ35_EINVAL, "paged prepare: position axes overlap");
  rc = check_heads("paged prepare: queries", q, rows, q_heads, cache->head_dim, false);
  if (!rc) rc = check_heads("paged prepare: keys", k, rows, cache->kv_heads, cache->head_dim, false);
  if (!rc) rc = check_heads("paged prepare: values", v, rows, cache->kv_heads, cache->head_dim, false);
  if (!rc) rc = check_heads("paged prepare: rotated queries", q_out, rows, q_heads, cache->head_dim, true);
  if (rc) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  OperatorDevice on;
  rc = on.enter({cache->keys, cache->values, q->data, k->data, v->data, q_weight, k_weight, inv_freq, positions, slots,
                 q_out->data}, s);
  if (rc) return rc;
  PrepareArgs a{};
  a.q = (const uint16_t*)q->data, a.q_row = q->row_stride, a.q_head = q->head_stride;
  a.k = (const uint16_t*)k->data, a.k_row = k->row_stride, a.k_head = k->head_stride;
  a.v = (const uint16_t*)v->data, a.v_row = v->row_stride, a.v_head = v->head_stride;
  a.out = (uint16_t*)q_out->data, a.out_row = q_out->row_stride, a.out_head = q_out->head_stride;
  a.keys = (uint16_t*)cache->keys, a.values = (uint16_t*)cache->values, a.pages = cache->pages;
  a.page_stride = cache->page_stride, a.row_stride = cache->row_stride, a.head_stride = cache->head_stride;
  a.shift = page_shift(cache->page_size), a.rows = rows, a.q_heads = q_heads, a.kv_heads = cache->kv_heads;
  a.rope_dim = rope_dim, a.q_weight = q_weight, a.k_weight = k_weight, a.eps = eps, a.inv_freq = inv_freq;
  a.positions = positions, a.position_stride = position_stride, a.slots = slots;
  if (pair_axis) memcpy(a.axis, pair_axis, (size_t)rope_dim / 2);
  a.tokens = (int)std::min<int64_t>(kPrepMostTokens, std::max<int64_t>(1, rows / kPrepBlocks));
  const dim3 grid((unsigned)((rows + a.tokens - 1) / a.tokens));
  auto kernel = cache->head_dim == 256 ? k_paged_prepare<256> : cache->head_dim == 128 ? k_paged_prepare<128> : k_paged_prepare<64>;
  return launch_operator("paged prepare", kernel, grid, kPrepThreads, 0, s, a);
}

namespace {

int check_attention_sizes(const char* what, int64_t rows, int64_t requests, int32_t q_heads, int32_t kv_heads,
                          int32_t head_dim, int64_t max_rows, int64_t max_keys) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(CQ35_EUNSUPPORTED, "%s: head_dim %d is not 64, 128 or 256", what, head_dim);
  if (kv_heads < 1 || kv_heads > 1024 || q_heads < 1 || q_heads > 4096 || q_heads % kv_heads)
    return fail(CQ35_EINVAL, "%s: %d query heads over %d key/value heads", what, q_heads, kv_heads);
  if (rows < 0 || requests < 0 || requests > kAttendMostRequests || max_rows < 0 || max_keys < 0 ||
      rows > INT32_MAX / (q_heads / kv_heads))
    return fail(CQ35_ERANGE, "%s: %lld rows of %lld requests, at most %lld rows and %lld keys each", what, (long long)rows,
                (long long)requests, (long long)max_rows, (long long)max_keys);
  const AttendPlan p = plan_attention(rows, requests, q_heads, kv_heads, head_dim, max_rows, max_keys);
  if (p.items > kMostBlocks || p.units > kMostBlocks)
    return fail(CQ35_ERANGE, "%s: too many rows for one call: %lld", what, (long long)rows);
  return CQ35_OK;
}

template <int HD>
int launch_attention(const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
  const AttendKernels k = attend_kernels<HD>(p);
  if (k.lds > 65536) HIP_TRY(hipFuncSetAttribute((const void*)k.attend, hipFuncAttributeMaxDynamicSharedMemorySize, (int)k.lds));
  int rc = launch_operator("paged attention", k.attend, k.grid, k.threads, k.lds, s, a);
  if (!rc && a.cut.slots > 0) rc = launch_operator("paged attention", k.join, k.join_grid, k.join_threads, 0, s, a);
  return rc;
}

}  // namespace

extern "C" int cq35_paged_attention_workspace(int64_t rows, int64_t requests, int32_t q_heads, int32_t kv_heads,
                                              int32_t head_dim, int64_t max_rows, int64_t max_keys, int64_t* bytes) {
  if (!bytes) return fail(CQ35_EINVAL, "paged attention workspace: null argument");
  const int rc = check_attention_sizes("paged attention workspace", rows, requests, q_heads, kv_heads, head_dim, max_rows, max_keys);
  if (rc) return rc;
  const AttendPlan p = plan_attention(rows, requests, q_heads, kv_heads, head_dim, max_rows, max_keys);
  *bytes = p.floats * (int64_t)sizeof(float);
  return CQ35_OK;
}

extern "C" int cq35_paged_attention(const cq35_paged_cache* cache, const cq35_heads* q, const cq35_heads* gate,
                                    const cq35_heads* out, int64_t rows, int32_t q_heads, const int32_t* table,
                                    int64_t table_stride, int64_t requests, int64_t width, const int32_t* row_start,
                                    const int32_t* lengths, float scale, int64_t max_rows, int64_t max_keys,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_cache(cache);
  if (!rc) rc = check_q_heads(cache, q_heads);
  if (!rc) rc = check_attention_sizes("paged attention", rows, requests, q_heads, cache->kv_heads, cache->head_dim, max_rows, max_keys);
  if (rc) return rc;
  if (rows == 0 || requests == 0) return CQ35_OK;
  if (!table || !row_start || !lengths) return fail(CQ35_EINVAL, "paged attention: null argument");
  if (width < 1 || width > (1 << 30) / cache->page_size || table_stride < 0)
    return fail(CQ35_ERANGE, "paged attention: tables of %lld pages", (long long)width);
  if (!std::isfinite(scale * 1.44269504f)) return fail(CQ35_EINVAL, "paged attention: scale %g", (double)scale);
  rc = check_heads("paged attention: queries", q, rows, q_heads, cache->head_dim, false);
  if (!rc && gate) rc = check_heads("paged attention: gate", gate, rows, q_heads, cache->head_dim, false);
  if (!rc) rc = check_heads("paged attention: output", out, rows, q_heads, cache->head_dim, true);
  if (rc) return rc;
  const AttendPlan p = plan_attention(rows, requests, q_heads, cache->kv_heads, cache->head_dim, max_rows, max_keys);
  const int64_t need = p.floats * (int64_t)sizeof(float);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(CQ35_EINVAL, "paged attention: %lld bytes of workspace at a 16-byte address needed, %lld given",
                (long long)need, (long long)(workspace ? workspace_bytes : 0));
  hipStream_t s = static_cast<hipStream_t>(stream);
  OperatorDevice on;
  rc = on.enter({cache->keys, cache->values, q->data, gate ? gate->data : nullptr, out->data, table, row_start, lengths,
                 need > 0 ? workspace : nullptr}, s);
  if (rc) return rc;
  AttendArgs a{};
  a.q = (const uint16_t*)q->data, a.q_row = q->row_stride, a.q_head = q->head_stride;
  if (gate) a.gate = (const uint16_t*)gate->data, a.gate_row = gate->row_stride, a.gate_head = gate->head_stride;
  a.out = (uint16_t*)out->data, a.out_row = out->row_stride, a.out_head = out->head_stride;
  a.keys = (const uint16_t*)cache->keys, a.values = (const uint16_t*)cache->values, a.pages = cache->pages;
  a.page_stride = cache->page_stride, a.row_stride = cache->row_stride, a.head_stride = cache->head_stride;
  a.shift = page_shift(cache->page_size), a.table = table, a.table_stride = table_stride;
  a.row_start = row_start, a.lengths = lengths, a.requests = (int)requests;
  a.cut = p.cut, a.cut.most_keys = (int32_t)(width * cache->page_size), a.part = static_cast<float*>(workspace);
  attend_scale(&a, scale);
  if (cache->head_dim == 256) return launch_attention<256>(a, p, s);
  if (cache->head_dim == 128) return launch_attention<128>(a, p, s);
  return launch_attention<64>(a, p, s);
}
