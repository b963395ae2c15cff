// Block tables and slot maps of one step, from the request lengths alone.
//
//   held  = ceil(length / 64)                      pages a request has
//   want  = ceil((length + added) / 64)            pages it needs; added < 0: the request ends
//
// Ended requests push their pages on the free stack (requests in order, pages in order); then the
// other requests, in order, pop `want - held` pages each from its top.  A request is admitted if
// its rows and pages fit and the stack holds what it and all earlier ones ask for; a request that
// is refused keeps its length.  Everything is a prefix sum over the requests, so the result does
// not depend on any order of execution.
//
// The work is small (8 bytes per row, 16 per run) and a launch costs more than it: ONE cluster of
// eight CTAs does the whole step.  Every CTA computes all prefix sums itself (a handful of block
// scans over at most 8192 requests) instead of waiting for another CTA's; one cluster barrier
// orders the step: before it all inputs are read, so that `lengths_out` may be `lengths`, and all pages
// are pushed; behind it pages are popped and the results written.  Slots are written run by run, a few
// runs to every warp of the cluster.  64 requests of one token: 5.6 us (6.3 with
// requests that end and inputs that are not in L2); 301 prompts with 57,000 rows: 8.4 us (14.9 with a search for
// every row).  A few small requests take one CTA.
#include <cooperative_groups.h>

#include "vsa_paged_common.cuh"

namespace vsa {

namespace {

namespace cg = cooperative_groups;

constexpr int kPlanThreads = 1024;
constexpr int kPlanCluster = 8;

struct RequestPlan {
  long long after;   // rows up to and including this request
  int runs_after;    // runs up to and including this request
  int taken;         // pages that earlier requests take, or -1: not admitted
  int length, given;  // tokens in the cache; pages that earlier requests give back
};

// Inclusive prefix sum over the block; `carry` is added and moved on to the next chunk.
template <typename T>
__device__ T block_scan(T x, T* warp_sums, T& carry) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const T y = __shfl_up_sync(~0u, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the previous scan's sums have been read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  T w = warp_sums[lane];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const T y = __shfl_up_sync(~0u, w, d);
    if (lane >= d) w += y;
  }
  const T before = __shfl_sync(~0u, w, warp == 0 ? 0 : warp - 1);
  const T all = __shfl_sync(~0u, w, 31);
  x += carry + (warp == 0 ? T(0) : before);
  carry += all;
  return x;
}

__device__ __forceinline__ int pages_of(long long tokens) { return static_cast<int>((tokens + kBlock - 1) / kBlock); }

template <int kCluster>
__device__ __forceinline__ void plan(const PagedPlanParams& p) {
  extern __shared__ __align__(16) char smem[];
  RequestPlan* plan = reinterpret_cast<RequestPlan*>(smem);
  __shared__ long long sums64[32];
  __shared__ int sums32[32];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, chunk_end = (p.requests + kPlanThreads - 1) / kPlanThreads * kPlanThreads;
  const int rank = kCluster > 1 ? static_cast<int>(cluster.block_rank()) : 0;

  // Rows and returned pages.
  long long rows_carry = 0;
  int back_carry = 0;
  for (int s = tid; s < chunk_end; s += kPlanThreads) {
    long long add = 0;
    int length = 0, back = 0;
    if (s < p.requests) {
      const int n = p.added[s];
      length = max(p.lengths[s], 0);
      add = max(n, 0);
      back = n < 0 ? min(pages_of(length), p.width) : 0;
    }
    const long long after = block_scan(add, sums64, rows_carry);
    const int back_after = block_scan(back, sums32, back_carry);
    if (s < p.requests) {
      plan[s].length = length;
      plan[s].after = p.rows_per_request > 0 ? static_cast<long long>(s) * p.rows_per_request + add : after;
      plan[s].given = back_after - back;
    }
  }
  const int count = min(max(*p.free_count, 0), p.pool);
  const int top = static_cast<int>(min(static_cast<long long>(count) + back_carry, static_cast<long long>(p.pool)));

  // Pages taken and runs.
  int need_carry = 0, runs_carry = 0, used = 0;
  for (int s = tid; s < chunk_end; s += kPlanThreads) {
    int need = 0, number = 0;
    bool fits = false;
    long long add = 0, total = 0;
    int length = 0;
    if (s < p.requests) {
      const int n = p.added[s];
      length = plan[s].length;
      add = max(n, 0);
      total = length + add;
      fits = n >= 0 && total <= static_cast<long long>(p.width) * kBlock && (add == 0 || plan[s].after <= p.tokens) &&
             (p.rows_per_request <= 0 || add <= p.rows_per_request);
      if (fits) need = pages_of(total) - pages_of(length);
    }
    const int taken = block_scan(need, sums32, need_carry);
    const bool admitted = fits && (need == 0 || taken <= top);
    if (admitted && add > 0) number = static_cast<int>((total - 1) / kBlock) - length / kBlock + 1;
    const int runs_after = block_scan(number, sums32, runs_carry);
    if (s < p.requests) {
      plan[s].taken = admitted ? taken - need : -1;
      plan[s].runs_after = runs_after;
      if (admitted) used = max(used, need > 0 ? taken : 0);
    }
  }
  // Admitted requests that need pages are a prefix of those that do: the largest sum is what is taken.
#pragma unroll
  for (int d = 16; d > 0; d /= 2) used = max(used, __shfl_xor_sync(~0u, used, d));
  __syncthreads();
  if ((tid & 31) == 0) sums32[tid >> 5] = used;
  __syncthreads();
  used = sums32[tid & 31];
#pragma unroll
  for (int d = 16; d > 0; d /= 2) used = max(used, __shfl_xor_sync(~0u, used, d));

  // Returned pages go on the stack.  Each warp of the cluster walks requests of its own.
  const int warp = (tid >> 5) * kCluster + rank,  // neighbours on different SMs
            warps = kCluster * (kPlanThreads / 32), lane = tid & 31;
  for (int s = warp; s < p.requests; s += warps) {
    if (p.added[s] >= 0) continue;
    const int held = min(pages_of(plan[s].length), p.width);
    for (int i = lane; i < held; i += 32) {
      const long long at = static_cast<long long>(count) + plan[s].given + i;
      if (at < p.pool) p.free_pages[at] = p.tables[s * p.table_stride + i];
    }
  }
  // Every input has been read, every page pushed.
  if (kCluster > 1) cluster.sync();
  else __syncthreads();

  // Behind the last request's rows and the last run.
  const long long thread = static_cast<long long>(rank) * kPlanThreads + tid, threads = kCluster * kPlanThreads;
  const long long rows_end = p.rows_per_request > 0 ? static_cast<long long>(p.requests) * p.rows_per_request : rows_carry;
  for (long long t = rows_end + thread; t < p.tokens; t += threads) p.row_slot[t] = -1;
  for (long long i = runs_carry + thread; i < p.max_runs; i += threads) p.runs[i] = make_int4(0, 0, 0, 0);
  for (int s = warp; s < p.requests; s += warps) {
    // Lane 0 reads before it writes: `lengths_out` may be `lengths`, `added` is never written.
    const RequestPlan r = plan[s];
    const int n = p.added[s];
    const long long total = r.length + static_cast<long long>(max(n, 0));
    if (lane == 0) {
      p.lengths_out[s] = n < 0 ? 0 : (r.taken >= 0 ? static_cast<int>(total) : r.length);
      p.admitted[s] = r.taken >= 0;
    }
    // Rows of the request that get no slot.
    const long long row0 = r.after - max(n, 0), taken_rows = r.taken >= 0 ? max(n, 0) : 0;
    const long long own_end = p.rows_per_request > 0 ? row0 + p.rows_per_request : r.after;
    for (long long t = row0 + taken_rows + lane; t < min(own_end, p.tokens); t += 32) p.row_slot[t] = -1;
    if (r.taken < 0) continue;
    const int held = pages_of(r.length), want = pages_of(total);
    for (int i = held + lane; i < want; i += 32)
      p.tables[s * p.table_stride + i] = p.free_pages[top - 1 - r.taken - (i - held)];
  }
  if (thread == 0) *p.free_count_out = top - used;

  // Up to 32 runs a warp at a time: a lane finds its run's request by binary search over the runs' prefix sums, then
  // the warp writes the slots of one run after the other.
  const int runs = min(runs_carry, p.max_runs);
  const int batch = min(max((runs + warps - 1) / warps, 4), 32);
  for (int base = warp * batch; base < runs; base += warps * batch) {
    const int at = base + lane;
    int4 run = make_int4(0, 0, 0, 0);
    if (lane < batch && at < runs) {
      int low = 0, high = p.requests - 1;  // first request with runs_after > at
      while (low < high) {
        const int mid = (low + high) / 2;
        if (plan[mid].runs_after > at) high = mid; else low = mid + 1;
      }
      const RequestPlan r = plan[low];
      const int n = p.added[low], begin = r.length / kBlock, held = pages_of(r.length);
      const long long total = r.length + static_cast<long long>(n), row0 = r.after - n;
      const int number = static_cast<int>((total - 1) / kBlock) - begin + 1, logical = begin + at - (r.runs_after - number);
      const long long first = max(static_cast<long long>(r.length), static_cast<long long>(logical) * kBlock);
      const long long last = min(total, (logical + 1LL) * kBlock);
      const int page = logical < held ? p.tables[low * p.table_stride + logical]
                                      : p.free_pages[top - 1 - r.taken - (logical - held)];
      run = make_int4(static_cast<int>(row0 + first - r.length), static_cast<int>(last - first), page,
                      static_cast<int>(first - static_cast<long long>(logical) * kBlock));
      p.runs[at] = run;
    }
    if (__reduce_max_sync(~0u, run.y) <= 4) {  // a decode step: a lane writes its own run's slots
      for (int t = 0; t < run.y; ++t) p.row_slot[run.x + t] = static_cast<int64_t>(run.z) * kBlock + run.w + t;
      continue;
    }
#pragma unroll 4
    for (int i = 0; i < batch; ++i) {
      const int row = __shfl_sync(~0u, run.x, i), count = __shfl_sync(~0u, run.y, i);
      const int64_t slot = static_cast<int64_t>(__shfl_sync(~0u, run.z, i)) * kBlock + __shfl_sync(~0u, run.w, i) + lane;
      if (lane < count) p.row_slot[row + lane] = slot;
      if (lane + 32 < count) p.row_slot[row + lane + 32] = slot + 32;
    }
  }
}

__global__ void __cluster_dims__(kPlanCluster, 1, 1) __launch_bounds__(kPlanThreads) paged_plan_cluster_kernel(PagedPlanParams p) { plan<kPlanCluster>(p); }
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const __grid_constant__ PagedPlanParams p) {
  pdl_wait();
  pdl_release();
  plan<1>(p);
}

}  // namespace

cudaError_t launch_paged_plan(const PagedPlanParams& p, cudaStream_t stream) {
  const int smem = p.requests * static_cast<int>(sizeof(RequestPlan));
  static_assert(kMaxRequests * sizeof(RequestPlan) <= 200 * 1024, "the requests' table fits shared memory");
  // One CTA : a cluster, us on the device.  Requests of one token: 1 request 4.6 : 5.2, 32 5.3 : 5.4, 64 5.6 : 5.7, 96
  // 6.4 : 5.9, 128 6.8 : 5.8, 256 8.9 : 6.4.  32 of 64 tokens 5.6 : 5.8, 64 of 32 tokens 6.1 : 5.9, 64 of 100 tokens
  // 6.8 : 5.8, 128 of 16 tokens 7.8 : 5.8.  At the limits the two are alike on the device; what decides there is the
  // host, whose call is 0.6 us shorter without a cluster (16.2 : 16.8).
  if (p.requests <= 64 && p.tokens <= 2048) return launch_overlapped<paged_plan_kernel>(dim3(1), kPlanThreads, smem, stream, p);
  const cudaError_t err = allow_shared<paged_plan_cluster_kernel>(smem);
  if (err != cudaSuccess) return err;
  paged_plan_cluster_kernel<<<kPlanCluster, kPlanThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace vsa
