// Internal launch interface of the paged key/value cache (plan, append, select, attention).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace vsa {

// Element types of the C entry points' `dtype` arguments.
enum PagedType : int { kBf16 = 0, kFp16 = 1, kE4m3 = 2 };

// Values written to the cache's status word, 0 = fine.
enum PagedError : int {
  kPagedBadPage = 200,  // a table named a page that the cache does not have: its tokens were left out
};

constexpr int kMostSelectPages = 24576;  // of one request: their 64-bit scores sit in shared memory
constexpr int kMaxRequests = 8192;   // of one step: the plan's per-request table sits in shared memory

struct PagedPlanParams {
  const int32_t* lengths;      // [requests] tokens in the cache
  const int32_t* added;        // [requests] new tokens, negative = the request ends
  int32_t* tables;             // [requests, width]
  long long table_stride;
  int width, requests;
  int32_t* free_pages;         // [pool] stack of free pages, `free_count` of them valid
  int pool;
  const int32_t* free_count;   // [1]
  long long tokens;            // rows of the step
  int rows_per_request;        // 0 = rows packed
  int32_t* lengths_out;        // [requests], may be `lengths`
  int32_t* free_count_out;     // [1], may be `free_count`
  uint8_t* admitted;           // [requests]
  int64_t* row_slot;           // [tokens]
  int4* runs;                  // [max_runs] {first row, rows, page, first row in the page}
  int max_runs;
};
cudaError_t launch_paged_plan(const PagedPlanParams& p, cudaStream_t stream);

struct PagedAppendParams {
  const void *k, *v;           // [tokens, kv_heads, 128] with strides in elements
  long long k_row_stride, k_head_stride, v_row_stride, v_head_stride;
  int dtype;
  long long tokens;
  void *k_cache, *v_cache;     // [pages, kv_heads, 64, 128]
  int cache_dtype;
  float *k_sum, *v_sum;        // [pages, kv_heads, 128]
  const float *k_scale, *v_scale;  // [kv_heads], 8-bit caches
  const int4* runs;
  int max_runs, pages, kv_heads;
  int* status;
};
cudaError_t launch_paged_append(const PagedAppendParams& p, cudaStream_t stream);

struct PagedSelectParams {
  const void* q;               // [requests, kv_heads * group, 128]
  long long q_row_stride, q_head_stride;
  int dtype;
  const float *k_sum, *v_sum;
  const int32_t* tables;
  long long table_stride;
  int width;
  const int32_t* lengths;
  int requests, kv_heads, group, pages, keep, first, last;
  float scale;
  int32_t* chosen;             // [requests, kv_heads, keep]
  float* coarse;               // [requests, kv_heads * group, 128] or null
  char* workspace;             // paged_select_workspace_bytes(...)
  bool early;                  // q, tables and lengths were complete before the preceding kernel began its work
  int* status;
};
int64_t paged_select_workspace_bytes(int requests, int kv_heads, int group, int width, bool choose, bool coarse);
cudaError_t launch_paged_select(const PagedSelectParams& p, cudaStream_t stream);

struct PagedAttentionParams {
  const void* q;
  long long q_row_stride, q_head_stride;
  int dtype;
  const void *k_cache, *v_cache;
  int cache_dtype;
  const float *k_scale, *v_scale;
  int pages;
  const int32_t* tables;
  long long table_stride;
  int width;
  const int32_t* lengths;
  int requests, kv_heads, group;
  const int32_t* chosen;       // [requests, kv_heads, keep] logical pages, -1 = none, or null = all pages
  int keep;
  const void* gate;            // [requests, kv_heads * group, 128] or null
  long long gate_row_stride, gate_head_stride;
  const float* coarse;
  float scale;
  void* out;                   // [requests, kv_heads * group, 128]
  float* lse;                  // [requests, kv_heads * group] or null
  float* workspace;            // paged_workspace_bytes(...)
  bool early;                  // as in PagedSelectParams
  int* status;
};
// `most_pages`: the table's width, or what is kept of it.
// Attention with one CTA to a tile: (request, key/value head) and up to eight query heads.
bool is_short_attention(int64_t tiles, int group, int most_pages, bool e4m3);
cudaError_t launch_paged_attention_short(const PagedAttentionParams& p, int most_pages, cudaStream_t stream);
// `tiles` = requests * key/value heads; `most_pages` a request can have or, if pages are chosen, choose.
int64_t paged_workspace_bytes(int64_t tiles, int group, int most_pages, bool e4m3);
int launch_paged_attention(const PagedAttentionParams& p, cudaStream_t stream);  // a Status

}  // namespace vsa
