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

constexpr int64_t kMostPages = 0x7fffffffLL / vsa::kBlock;

}  // namespace

extern "C" {

int vsa_paged_plan(const int32_t* lengths, const int32_t* added, int32_t* tables, int64_t table_stride, int32_t width,
                   int32_t requests, int32_t* free_pages, int32_t pool, const int32_t* free_count, int64_t tokens,
                   int32_t rows_per_request, int32_t* lengths_out, int32_t* free_count_out, uint8_t* admitted,
                   int64_t* row_slot, int32_t* runs, int32_t max_runs, void* stream) {
  if (lengths == nullptr || added == nullptr || tables == nullptr || free_pages == nullptr || free_count == nullptr ||
      lengths_out == nullptr || free_count_out == nullptr || admitted == nullptr || row_slot == nullptr ||
      runs == nullptr || misaligned(runs) || requests <= 0 || width <= 0 || table_stride < width || pool <= 0 ||
      tokens <= 0 || rows_per_request < 0 || max_runs <= 0)
    return vsa::kBadArgument;
  if (requests > vsa::kMaxRequests || tokens > 0x7fffffffLL || width > kMostPages ||
      static_cast<int64_t>(requests) * width > 0x7fffffffLL)
    return vsa::kTooLarge;
  vsa::PagedPlanParams p{};
  p.lengths = lengths;
  p.added = added;
  p.tables = tables;
  p.table_stride = table_stride;
  p.width = width;
  p.requests = requests;
  p.free_pages = free_pages;
  p.pool = pool;
  p.free_count = free_count;
  p.tokens = tokens;
  p.rows_per_request = rows_per_request;
  p.lengths_out = lengths_out;
  p.free_count_out = free_count_out;
  p.admitted = admitted;
  p.row_slot = row_slot;
  p.runs = reinterpret_cast<int4*>(runs);
  p.max_runs = max_runs;
  return from_cuda(vsa::launch_paged_plan(p, as_stream(stream)));
}

int vsa_paged_append(const void* k, const void* v, int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
                     int64_t v_head_stride, int32_t dtype, int64_t tokens, void* k_cache, void* v_cache,
                     int32_t cache_dtype, float* k_sum, float* v_sum, const float* k_scale, const float* v_scale,
                     const int32_t* runs, int32_t max_runs, int32_t pages, int32_t kv_heads, int32_t* status,
                     void* stream) {
  if (k == nullptr || v == nullptr || k_cache == nullptr || v_cache == nullptr || k_sum == nullptr ||
      v_sum == nullptr || runs == nullptr || misaligned(k, v, k_cache, v_cache) || misaligned(runs) ||
      bad_strides(k_row_stride, k_head_stride) || bad_strides(v_row_stride, v_head_stride) || tokens <= 0 ||
      max_runs <= 0 || pages <= 0 || kv_heads <= 0 || (dtype != vsa::kBf16 && dtype != vsa::kFp16) ||
      (cache_dtype != dtype && cache_dtype != vsa::kE4m3) ||
      (cache_dtype == vsa::kE4m3 && (k_scale == nullptr || v_scale == nullptr)))
    return vsa::kBadArgument;
  if (kv_heads > 65535 || static_cast<int64_t>(pages) * kv_heads > kMostPages) return vsa::kTooLarge;
  vsa::PagedAppendParams p{};
  p.k = k;
  p.v = v;
  p.k_row_stride = k_row_stride;
  p.k_head_stride = k_head_stride;
  p.v_row_stride = v_row_stride;
  p.v_head_stride = v_head_stride;
  p.dtype = dtype;
  p.tokens = tokens;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.cache_dtype = cache_dtype;
  p.k_sum = k_sum;
  p.v_sum = v_sum;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.runs = reinterpret_cast<const int4*>(runs);
  p.max_runs = max_runs;
  p.pages = pages;
  p.kv_heads = kv_heads;
  p.status = status;
  return from_cuda(vsa::launch_paged_append(p, as_stream(stream)));
}

static int select_common(const void* q, int64_t q_row_stride, int64_t q_head_stride, int32_t dtype, const float* k_sum,
                     const float* v_sum, const int32_t* tables, int64_t table_stride, int32_t width,
                     const int32_t* lengths, int32_t requests, int32_t kv_heads, int32_t group, int32_t pages,
                     int32_t keep, int32_t first, int32_t last, float scale, int32_t* chosen, float* coarse,
                     void* workspace, int64_t workspace_bytes, int32_t* status, void* stream, bool early) {
  if (q == nullptr || k_sum == nullptr || v_sum == nullptr || tables == nullptr || lengths == nullptr ||
      (chosen == nullptr && coarse == nullptr) || misaligned(q, k_sum, v_sum, coarse) ||
      bad_strides(q_row_stride, q_head_stride) || (dtype != vsa::kBf16 && dtype != vsa::kFp16) || width <= 0 ||
      table_stride < width || requests <= 0 || kv_heads <= 0 || group <= 0 || pages <= 0 || first < 0 || last < 0 ||
      (chosen != nullptr && (keep <= 0 || keep - first < last)))
    return vsa::kBadArgument;
  // One request's scores must fit the shared memory of a CTA.
  if ((chosen != nullptr && width > vsa::kMostSelectPages) || width > kMostPages ||
      static_cast<int64_t>(pages) * kv_heads > kMostPages ||
      requests > vsa::kMaxRequests || static_cast<int64_t>(requests) * width * kv_heads * group > 0x7fffffffLL)
    return vsa::kTooLarge;
  if (workspace == nullptr || misaligned(workspace) ||
      workspace_bytes < vsa_paged_select_workspace_bytes(requests, kv_heads, group, width, chosen != nullptr, coarse != nullptr))
    return vsa::kBadArgument;
  vsa::PagedSelectParams p{};
  p.q = q;
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.dtype = dtype;
  p.k_sum = k_sum;
  p.v_sum = v_sum;
  p.tables = tables;
  p.table_stride = table_stride;
  p.width = width;
  p.lengths = lengths;
  p.requests = requests;
  p.kv_heads = kv_heads;
  p.group = group;
  p.pages = pages;
  p.keep = keep;
  p.first = first;
  p.last = last;
  p.scale = scale;
  p.chosen = chosen;
  p.coarse = coarse;
  p.workspace = static_cast<char*>(workspace);
  p.early = early;
  p.status = status;
  return from_cuda(vsa::launch_paged_select(p, as_stream(stream)));
}

int vsa_paged_select(const void* q, int64_t q_row_stride, int64_t q_head_stride, int32_t dtype, const float* k_sum,
                     const float* v_sum, const int32_t* tables, int64_t table_stride, int32_t width,
                     const int32_t* lengths, int32_t requests, int32_t kv_heads, int32_t group, int32_t pages,
                     int32_t keep, int32_t first, int32_t last, float scale, int32_t* chosen, float* coarse,
                     void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  return select_common(q, q_row_stride, q_head_stride, dtype, k_sum, v_sum, tables, table_stride, width, lengths, requests,
                       kv_heads, group, pages, keep, first, last, scale, chosen, coarse, workspace, workspace_bytes, status,
                       stream, false);
}

static int attention_common(const void* q, int64_t q_row_stride, int64_t q_head_stride, int32_t dtype,
                        const void* k_cache, const void* v_cache, int32_t cache_dtype, const float* k_scale,
                        const float* v_scale, int32_t pages, const int32_t* tables, int64_t table_stride,
                        int32_t width, const int32_t* lengths, int32_t requests, int32_t kv_heads, int32_t group,
                        const int32_t* chosen, int32_t keep, const void* gate, int64_t gate_row_stride,
                        int64_t gate_head_stride, const float* coarse, float scale, void* out, float* lse,
                        void* workspace, int64_t workspace_bytes, int32_t* status, void* stream, bool early) {
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || tables == nullptr || lengths == nullptr ||
      out == nullptr || misaligned(q, k_cache, v_cache, out) || misaligned(gate, coarse, workspace) ||
      bad_strides(q_row_stride, q_head_stride) || (dtype != vsa::kBf16 && dtype != vsa::kFp16) ||
      (cache_dtype != dtype && cache_dtype != vsa::kE4m3) ||
      (cache_dtype == vsa::kE4m3 && (k_scale == nullptr || v_scale == nullptr)) || width <= 0 ||
      table_stride < width || requests <= 0 || kv_heads <= 0 || group <= 0 || pages <= 0 ||
      (chosen != nullptr && keep <= 0) ||
      (gate != nullptr && (coarse == nullptr || bad_strides(gate_row_stride, gate_head_stride))))
    return vsa::kBadArgument;
  const int64_t need = vsa_paged_workspace_bytes(group, chosen == nullptr || keep > width ? width : keep);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return vsa::kBadArgument;
  if (static_cast<int64_t>(pages) * kv_heads > kMostPages || width > kMostPages ||
      requests > vsa::kMaxRequests || static_cast<int64_t>(requests) * width * kv_heads * group > 0x7fffffffLL)
    return vsa::kTooLarge;
  vsa::PagedAttentionParams p{};
  p.q = q;
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.dtype = dtype;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.cache_dtype = cache_dtype;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.pages = pages;
  p.tables = tables;
  p.table_stride = table_stride;
  p.width = width;
  p.lengths = lengths;
  p.requests = requests;
  p.kv_heads = kv_heads;
  p.group = group;
  p.chosen = chosen;
  p.keep = keep;
  p.gate = gate;
  p.gate_row_stride = gate_row_stride;
  p.gate_head_stride = gate_head_stride;
  p.coarse = coarse;
  p.scale = scale;
  p.out = out;
  p.lse = lse;
  p.workspace = static_cast<float*>(workspace);
  p.early = early;
  p.status = status;
  return vsa::launch_paged_attention(p, as_stream(stream));
}

int vsa_paged_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, int32_t dtype,
                        const void* k_cache, const void* v_cache, int32_t cache_dtype, const float* k_scale,
                        const float* v_scale, int32_t pages, const int32_t* tables, int64_t table_stride,
                        int32_t width, const int32_t* lengths, int32_t requests, int32_t kv_heads, int32_t group,
                        const int32_t* chosen, int32_t keep, const void* gate, int64_t gate_row_stride,
                        int64_t gate_head_stride, const float* coarse, float scale, void* out, float* lse,
                        void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  return attention_common(q, q_row_stride, q_head_stride, dtype, k_cache, v_cache, cache_dtype, k_scale, v_scale, pages,
                          tables, table_stride, width, lengths, requests, kv_heads, group, chosen, keep, gate,
                          gate_row_stride, gate_head_stride, coarse, scale, out, lse, workspace, workspace_bytes, status,
                          stream, false);
}

int64_t vsa_paged_select_workspace_bytes(int32_t requests, int32_t kv_heads, int32_t group, int32_t width,
                                         int32_t choose, int32_t coarse) {
  return vsa::paged_select_workspace_bytes(requests, kv_heads, group, width, choose != 0, coarse != 0);
}

int64_t vsa_paged_workspace_bytes(int32_t group, int32_t most_pages) {
  return vsa::paged_workspace_bytes(group, most_pages);
}

namespace {

// Byte offsets in the workspace of a decode step.
struct DecodeSpace {
  int64_t coarse, select, attention, bytes;
};
DecodeSpace decode_space(int64_t requests, int64_t kv_heads, int32_t group, int32_t width, int64_t keep, bool gated) {
  const auto round = [](int64_t n) { return (n + 255) / 256 * 256; };
  DecodeSpace w{};
  w.coarse = round(requests * kv_heads * keep * 4);
  w.select = w.coarse + (gated ? round(requests * kv_heads * group * vsa::kDim * 4) : 0);
  const bool any = keep > 0 || gated;
  w.attention = w.select + (any ? round(vsa_paged_select_workspace_bytes(static_cast<int32_t>(requests), static_cast<int32_t>(kv_heads),
                                                                         group, width, keep > 0, gated)) : 0);
  w.bytes = w.attention + vsa_paged_workspace_bytes(group, keep > 0 && keep < width ? static_cast<int32_t>(keep) : width);
  if (w.bytes == 0) w.bytes = 16;
  return w;
}

}  // namespace

int64_t vsa_paged_decode_workspace_bytes(int32_t requests, int32_t kv_heads, int32_t group, int32_t width,
                                         int32_t keep, int32_t gated) {
  return decode_space(requests, kv_heads, group, width, keep, gated != 0).bytes;
}

int vsa_paged_decode(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k, const void* v,
                     int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                     int32_t dtype, int64_t tokens, void* k_cache, void* v_cache, int32_t cache_dtype, float* k_sum,
                     float* v_sum, const float* k_scale, const float* v_scale, int32_t pages, int32_t kv_heads,
                     int32_t group, const int32_t* runs, int32_t max_runs, const int32_t* tables, int64_t table_stride,
                     int32_t width, const int32_t* lengths, int32_t requests, int32_t keep, int32_t first, int32_t last,
                     const void* gate, int64_t gate_row_stride, int64_t gate_head_stride, float scale, void* out,
                     void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  if (requests <= 0 || kv_heads <= 0 || group <= 0 || width <= 0 || keep < 0 || workspace == nullptr || misaligned(workspace))
    return vsa::kBadArgument;
  const bool gated = gate != nullptr;
  const DecodeSpace w = decode_space(requests, kv_heads, group, width, keep, gated);
  if (workspace_bytes < w.bytes) return vsa::kBadArgument;
  char* base = static_cast<char*>(workspace);
  int32_t* chosen = keep > 0 ? reinterpret_cast<int32_t*>(base) : nullptr;
  float* coarse = gated ? reinterpret_cast<float*>(base + w.coarse) : nullptr;
  int rc = vsa_paged_append(k, v, k_row_stride, k_head_stride, v_row_stride, v_head_stride, dtype, tokens, k_cache, v_cache,
                            cache_dtype, k_sum, v_sum, k_scale, v_scale, runs, max_runs, pages, kv_heads, status, stream);
  if (rc == vsa::kOk && (keep > 0 || gated))
    rc = select_common(q, q_row_stride, q_head_stride, dtype, k_sum, v_sum, tables, table_stride, width, lengths, requests,
                       kv_heads, group, pages, keep, first, last, scale, chosen, coarse, base + w.select,
                       w.attention - w.select, status, stream, true);
  if (rc == vsa::kOk)
    rc = attention_common(q, q_row_stride, q_head_stride, dtype, k_cache, v_cache, cache_dtype, k_scale, v_scale, pages,
                          tables, table_stride, width, lengths, requests, kv_heads, group, chosen, keep, gate,
                          gate_row_stride, gate_head_stride, coarse, scale, out, nullptr, base + w.attention,
                          w.bytes - w.attention, status, stream, true);
  return rc;
}

}  // extern "C"
