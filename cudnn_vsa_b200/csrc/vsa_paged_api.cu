// extern "C" entry points of the paged key/value cache: argument checks and launches.
#include "../../include/vsa_b200.h"
#include "vsa_common.cuh"
#include "vsa_paged.h"

namespace {

int from_cuda(cudaError_t err) { return err == cudaSuccess ? vsa::kOk : vsa::kCudaError; }
cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }
bool misaligned(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) |
           reinterpret_cast<uintptr_t>(d)) & 15) != 0;
}
// Rows are read in 16-byte units.
bool bad_strides(int64_t row, int64_t head) { return row < 0 || head < 0 || row % 8 != 0 || head % 8 != 0; }

// Whether all values are in [least, 2^31).
template <class... Values>
bool in_range(int64_t least, Values... values) {
  return ((values >= least && values <= 0x7fffffffLL) && ...);
}
// a * b * ... < 2^31 for positive factors below 2^31.
template <class... Values>
bool small_product(Values... values) {
  int64_t product = 1;
  return ((product <= 0x7fffffffLL && (product *= values, product <= 0x7fffffffLL)) && ...);
}

// Units of work - (request, key/value head, up to eight of its query heads, page) - and query rows are numbered by
// 32-bit integers; so are a request's tokens and the rows of the cache.
bool too_large(int64_t requests, int64_t width, int64_t kv_heads, int64_t group, int64_t pages) {
  return requests > vsa::kMaxRequests || !small_product(pages, kv_heads, vsa::kBlock) || !small_product(width, vsa::kBlock) ||
         !small_product(requests, width, kv_heads, (group + 7) / 8) || !small_product(requests, kv_heads, group);
}

bool bad_types(int64_t dtype, int64_t cache_dtype, const void* k_scale, const void* v_scale) {
  return (dtype != vsa::kBf16 && dtype != vsa::kFp16) || (cache_dtype != dtype && cache_dtype != vsa::kE4m3) ||
         (cache_dtype == vsa::kE4m3 && (k_scale == nullptr || v_scale == nullptr));
}

int run_append(const vsa_paged_append_args& a) {
  if (a.k == nullptr || a.v == nullptr || a.k_cache == nullptr || a.v_cache == nullptr || a.k_sum == nullptr ||
      a.v_sum == nullptr || a.runs == nullptr || misaligned(a.k, a.v, a.k_cache, a.v_cache) || misaligned(a.runs) ||
      bad_strides(a.k_row_stride, a.k_head_stride) || bad_strides(a.v_row_stride, a.v_head_stride) ||
      !in_range(1, a.tokens, a.max_runs, a.pages, a.kv_heads) || bad_types(a.dtype, a.cache_dtype, a.k_scale, a.v_scale))
    return vsa::kBadArgument;
  if (a.kv_heads > 65535 || !small_product(a.pages, a.kv_heads, vsa::kBlock)) return vsa::kTooLarge;
  vsa::PagedAppendParams p{};
  p.k = a.k;
  p.v = a.v;
  p.k_row_stride = a.k_row_stride;
  p.k_head_stride = a.k_head_stride;
  p.v_row_stride = a.v_row_stride;
  p.v_head_stride = a.v_head_stride;
  p.dtype = static_cast<int>(a.dtype);
  p.tokens = a.tokens;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.cache_dtype = static_cast<int>(a.cache_dtype);
  p.k_sum = a.k_sum;
  p.v_sum = a.v_sum;
  p.k_scale = a.k_scale;
  p.v_scale = a.v_scale;
  p.runs = reinterpret_cast<const int4*>(a.runs);
  p.max_runs = static_cast<int>(a.max_runs);
  p.pages = static_cast<int>(a.pages);
  p.kv_heads = static_cast<int>(a.kv_heads);
  p.status = a.status;
  return from_cuda(vsa::launch_paged_append(p, as_stream(a.stream)));
}

// `early`: see PagedSelectParams.  Without `launch` the arguments are checked only.
int run_select(const vsa_paged_select_args& a, bool early, bool launch = true) {
  const bool choose = a.chosen != nullptr;
  if (a.q == nullptr || a.k_sum == nullptr || a.v_sum == nullptr || a.tables == nullptr || a.lengths == nullptr ||
      (!choose && a.coarse == nullptr) || misaligned(a.q, a.k_sum, a.v_sum, a.coarse) ||
      bad_strides(a.q_row_stride, a.q_head_stride) || bad_types(a.dtype, a.dtype, nullptr, nullptr) ||
      !in_range(1, a.width, a.requests, a.kv_heads, a.group, a.pages) || !in_range(0, a.keep, a.first, a.last) ||
      a.table_stride < a.width || (choose && (a.keep == 0 || a.keep - a.first < a.last)))
    return vsa::kBadArgument;
  // One request's scores must fit the shared memory of a CTA.
  if ((choose && a.width > vsa::kMostSelectPages) || too_large(a.requests, a.width, a.kv_heads, a.group, a.pages)) return vsa::kTooLarge;
  vsa::PagedSelectParams p{};
  p.q = a.q;
  p.q_row_stride = a.q_row_stride;
  p.q_head_stride = a.q_head_stride;
  p.dtype = static_cast<int>(a.dtype);
  p.k_sum = a.k_sum;
  p.v_sum = a.v_sum;
  p.tables = a.tables;
  p.table_stride = a.table_stride;
  p.width = static_cast<int>(a.width);
  p.lengths = a.lengths;
  p.requests = static_cast<int>(a.requests);
  p.kv_heads = static_cast<int>(a.kv_heads);
  p.group = static_cast<int>(a.group);
  p.pages = static_cast<int>(a.pages);
  p.keep = static_cast<int>(a.keep);
  p.first = static_cast<int>(a.first);
  p.last = static_cast<int>(a.last);
  p.scale = static_cast<float>(a.scale);
  p.chosen = a.chosen;
  p.coarse = a.coarse;
  p.workspace = static_cast<char*>(a.workspace);
  p.early = early;
  p.status = a.status;
  const int64_t need = vsa::paged_select_workspace_bytes(p.requests, p.kv_heads, p.group, p.width, choose, a.coarse != nullptr);
  if (need > 0 && (a.workspace == nullptr || misaligned(a.workspace) || a.workspace_bytes < need)) return vsa::kBadArgument;
  return launch ? from_cuda(vsa::launch_paged_select(p, as_stream(a.stream))) : vsa::kOk;
}

int run_attention(const vsa_paged_attention_args& a, bool early, bool launch = true) {
  if (a.q == nullptr || a.k_cache == nullptr || a.v_cache == nullptr || a.tables == nullptr || a.lengths == nullptr ||
      a.out == nullptr || misaligned(a.q, a.k_cache, a.v_cache, a.out) || misaligned(a.gate, a.coarse, a.workspace) ||
      bad_strides(a.q_row_stride, a.q_head_stride) || bad_types(a.dtype, a.cache_dtype, a.k_scale, a.v_scale) ||
      !in_range(1, a.width, a.requests, a.kv_heads, a.group, a.pages) || !in_range(0, a.keep) ||
      a.table_stride < a.width || (a.chosen != nullptr && a.keep == 0) ||
      (a.gate != nullptr && (a.coarse == nullptr || bad_strides(a.gate_row_stride, a.gate_head_stride))))
    return vsa::kBadArgument;
  if (too_large(a.requests, a.width, a.kv_heads, a.group, a.pages)) return vsa::kTooLarge;
  vsa::PagedAttentionParams p{};
  p.q = a.q;
  p.q_row_stride = a.q_row_stride;
  p.q_head_stride = a.q_head_stride;
  p.dtype = static_cast<int>(a.dtype);
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.cache_dtype = static_cast<int>(a.cache_dtype);
  p.k_scale = a.k_scale;
  p.v_scale = a.v_scale;
  p.pages = static_cast<int>(a.pages);
  p.tables = a.tables;
  p.table_stride = a.table_stride;
  p.width = static_cast<int>(a.width);
  p.lengths = a.lengths;
  p.requests = static_cast<int>(a.requests);
  p.kv_heads = static_cast<int>(a.kv_heads);
  p.group = static_cast<int>(a.group);
  p.chosen = a.chosen;
  p.keep = static_cast<int>(a.keep);
  p.gate = a.gate;
  p.gate_row_stride = a.gate_row_stride;
  p.gate_head_stride = a.gate_head_stride;
  p.coarse = a.coarse;
  p.scale = static_cast<float>(a.scale);
  p.out = a.out;
  p.lse = a.lse;
  p.workspace = static_cast<float*>(a.workspace);
  p.early = early;
  p.status = a.status;
  const int64_t need = vsa::paged_workspace_bytes(a.requests * a.kv_heads, p.group, p.chosen == nullptr || p.keep > p.width ? p.width : p.keep,
                                                  p.cache_dtype == vsa::kE4m3);
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need)) return vsa::kBadArgument;
  return launch ? vsa::launch_paged_attention(p, as_stream(a.stream)) : vsa::kOk;
}

// Byte offsets in the workspace of a decode step.
struct DecodeSpace {
  int64_t coarse, select, attention, bytes;
};
DecodeSpace decode_space(int64_t requests, int64_t kv_heads, int32_t group, int32_t width, int64_t keep, bool gated, bool e4m3) {
  const auto round = [](int64_t n) { return (n + 255) / 256 * 256; };
  DecodeSpace w{};
  w.coarse = round(requests * kv_heads * keep * 4);
  w.select = w.coarse + (gated ? round(requests * kv_heads * group * vsa::kDim * 4) : 0);
  w.attention = w.select;
  if (keep > 0 || gated)
    w.attention += round(vsa::paged_select_workspace_bytes(static_cast<int>(requests), static_cast<int>(kv_heads), group, width,
                                                           keep > 0, gated));
  w.bytes = w.attention + vsa::paged_workspace_bytes(requests * kv_heads, group, keep > 0 && keep < width ? static_cast<int>(keep) : width, e4m3);
  if (w.bytes == 0) w.bytes = 16;
  return w;
}

// A binding packs the structs as consecutive 64-bit fields.
static_assert(sizeof(vsa_paged_plan_args) == 18 * 8 && sizeof(vsa_paged_append_args) == 21 * 8 &&
                  sizeof(vsa_paged_select_args) == 24 * 8 && sizeof(vsa_paged_attention_args) == 30 * 8 &&
                  sizeof(vsa_paged_decode_args) == 40 * 8,
              "every field has 64 bits");

}  // namespace

extern "C" {

int vsa_paged_plan(const vsa_paged_plan_args* args) {
  if (args == nullptr) return vsa::kBadArgument;
  const vsa_paged_plan_args& a = *args;
  if (a.lengths == nullptr || a.added == nullptr || a.tables == nullptr || a.free_pages == nullptr ||
      a.free_count == nullptr || a.lengths_out == nullptr || a.free_count_out == nullptr || a.admitted == nullptr ||
      a.row_slot == nullptr || a.runs == nullptr || misaligned(a.runs) ||
      !in_range(1, a.width, a.requests, a.pool, a.tokens, a.max_runs) || !in_range(0, a.rows_per_request) ||
      a.table_stride < a.width)
    return vsa::kBadArgument;
  if (a.requests > vsa::kMaxRequests || !small_product(a.width, vsa::kBlock) || !small_product(a.requests, a.width))
    return vsa::kTooLarge;
  // A run that found no room in the list would leave its rows without slots, and their request admitted.
  if (a.max_runs < a.tokens && a.max_runs < a.tokens / vsa::kBlock + 2 * a.requests) return vsa::kBadArgument;
  vsa::PagedPlanParams p{};
  p.lengths = a.lengths;
  p.added = a.added;
  p.tables = a.tables;
  p.table_stride = a.table_stride;
  p.width = static_cast<int>(a.width);
  p.requests = static_cast<int>(a.requests);
  p.free_pages = a.free_pages;
  p.pool = static_cast<int>(a.pool);
  p.free_count = a.free_count;
  p.tokens = a.tokens;
  p.rows_per_request = static_cast<int>(a.rows_per_request);
  p.lengths_out = a.lengths_out;
  p.free_count_out = a.free_count_out;
  p.admitted = a.admitted;
  p.row_slot = a.row_slot;
  p.runs = reinterpret_cast<int4*>(a.runs);
  p.max_runs = static_cast<int>(a.max_runs);
  return from_cuda(vsa::launch_paged_plan(p, as_stream(a.stream)));
}

int vsa_paged_append(const vsa_paged_append_args* args) {
  return args == nullptr ? vsa::kBadArgument : run_append(*args);
}

int64_t vsa_paged_select_workspace_bytes(int32_t requests, int32_t kv_heads, int32_t group, int32_t width,
                                         int32_t choose, int32_t coarse) {
  return vsa::paged_select_workspace_bytes(requests, kv_heads, group, width, choose != 0, coarse != 0);
}

int vsa_paged_select(const vsa_paged_select_args* args) {
  return args == nullptr ? vsa::kBadArgument : run_select(*args, false);
}

int64_t vsa_paged_workspace_bytes(int32_t requests, int32_t kv_heads, int32_t group, int32_t most_pages,
                                  int32_t cache_dtype) {
  return vsa::paged_workspace_bytes(static_cast<int64_t>(requests) * kv_heads, group, most_pages, cache_dtype == vsa::kE4m3);
}

int vsa_paged_attention(const vsa_paged_attention_args* args) {
  return args == nullptr ? vsa::kBadArgument : run_attention(*args, false);
}

int64_t vsa_paged_decode_workspace_bytes(int32_t requests, int32_t kv_heads, int32_t group, int32_t width,
                                         int32_t keep, int32_t gated, int32_t cache_dtype) {
  return decode_space(requests, kv_heads, group, width, keep, gated != 0, cache_dtype == vsa::kE4m3).bytes;
}

int vsa_paged_decode(const vsa_paged_decode_args* args) {
  if (args == nullptr) return vsa::kBadArgument;
  const vsa_paged_decode_args& a = *args;
  if (!in_range(1, a.requests, a.kv_heads, a.group, a.width) || !in_range(0, a.keep) || a.workspace == nullptr ||
      misaligned(a.workspace))
    return vsa::kBadArgument;
  const bool gated = a.gate != nullptr, select = a.keep > 0 || gated;
  if (too_large(a.requests, a.width, a.kv_heads, a.group, 1)) return vsa::kTooLarge;  // `pages` is checked with the rest
  const DecodeSpace w = decode_space(a.requests, a.kv_heads, static_cast<int32_t>(a.group), static_cast<int32_t>(a.width), a.keep, gated,
                                     a.cache_dtype == vsa::kE4m3);
  if (a.workspace_bytes < w.bytes) return vsa::kBadArgument;
  char* base = static_cast<char*>(a.workspace);
  int32_t* chosen = a.keep > 0 ? reinterpret_cast<int32_t*>(base) : nullptr;
  float* coarse = gated ? reinterpret_cast<float*>(base + w.coarse) : nullptr;
  const vsa_paged_append_args append{a.k, a.v, a.k_row_stride, a.k_head_stride, a.v_row_stride, a.v_head_stride, a.dtype,
                                     a.tokens, a.k_cache, a.v_cache, a.cache_dtype, a.k_sum, a.v_sum, a.k_scale, a.v_scale,
                                     a.runs, a.max_runs, a.pages, a.kv_heads, a.status, a.stream};
  const vsa_paged_select_args choice{a.q, a.q_row_stride, a.q_head_stride, a.dtype, a.k_sum, a.v_sum, a.tables,
                                     a.table_stride, a.width, a.lengths, a.requests, a.kv_heads, a.group, a.pages, a.keep,
                                     a.first, a.last, a.scale, chosen, coarse, base + w.select, w.attention - w.select,
                                     a.status, a.stream};
  const vsa_paged_attention_args attention{a.q, a.q_row_stride, a.q_head_stride, a.dtype, a.k_cache, a.v_cache,
                                           a.cache_dtype, a.k_scale, a.v_scale, a.pages, a.tables, a.table_stride, a.width,
                                           a.lengths, a.requests, a.kv_heads, a.group, chosen, a.keep, a.gate,
                                           a.gate_row_stride, a.gate_head_stride, coarse, a.scale, a.out, nullptr,
                                           base + w.attention, w.bytes - w.attention, a.status, a.stream};
  // Nothing is enqueued unless all of it can be.
  int rc = select ? run_select(choice, true, false) : vsa::kOk;
  if (rc == vsa::kOk) rc = run_attention(attention, true, false);
  if (rc == vsa::kOk) rc = run_append(append);
  if (rc == vsa::kOk && select) rc = run_select(choice, true);
  if (rc == vsa::kOk) rc = run_attention(attention, true);
  return rc;
}

}  // extern "C"
