// Page selection for one new token per request, and the attention over the page means.
//
//   score[p]  = (sum over the group's query heads of q) . k_sum[p] / n_p       one per key/value head
//   chosen    = the first `first` and last `last` pages, and the highest scores up to `keep` in all
//   coarse_g  = softmax_p(scale * q_g . k_sum[p] / n_p) @ (v_sum[p] / n_p)      one per query head
//
// with n_p the tokens of page p (64, fewer in a request's last page).  Scores are formed in 64
// bits: a choice is a whole number, and with FP32 sums two pages whose scores differ by less than
// the rounding of a 128-term sum would be chosen by the order of the additions.  The pages' sums
// are read once (512 bytes per page and head, twice that with the coarse branch) and bound the
// kernels; the 64-bit products ride along.
//
//   page_scores_kernel  Warps are the workers: each takes the same count of consecutive pages of the
//                       (request, head) tiles and keeps its results to itself - a tile's running
//                       maximum, sum and output in registers - so that no warp waits for another.
//                       Its pages' sums arrive by cp.async in a ring of its own, two pages a step and
//                       kSteps steps deep (16 KiB a warp, 192 KiB an SM), half a warp to a page.  Every lane
//                       reads what it has copied itself, so that waiting for its own copies is enough.
//                       Incomplete tiles go to the workspace.
//   page_choose_kernel  Joins the incomplete tiles, one warp each, and chooses the pages, one CTA per
//                       (request, head): the interval that holds the last score kept is narrowed with
//                       histograms of 2048 equal bins over [lowest, highest candidate] - scores of
//                       real inputs are spread, so the first pass leaves a few candidates - and the pages
//                       are listed in ascending order.
#include "vsa_paged_common.cuh"

namespace vsa {

namespace {

constexpr int kScoreWarps = 12, kScoreThreads = 32 * kScoreWarps;
constexpr int kWorkersMax = 160 * kScoreWarps;
constexpr int kSteps = 8;                 // of two pages in flight per warp
constexpr int kLeastUnits = 4;            // pages a worker takes at least
constexpr int kColumnsMax = 4;            // query heads that share one pass over the sums
constexpr int kChooseThreads = 512, kChooseWarps = kChooseThreads / 32;
constexpr int kBins = 2048;
constexpr double kTopScore = 1e200;  // stands for +infinity and NaN: above every finite score

struct SelectParams {
  PagedSelectParams p;
  int chunks, chunk_heads;  // a group is taken in `chunks` parts of up to `chunk_heads` query heads
  int workers;
  double* score;            // [requests, kv_heads, width]
  float* partials;          // [2 * workers][chunk_heads][128]
  float2* stats;            // [2 * workers][chunk_heads]
  int4* split;              // [workers] {request, virtual head, last worker, 1} of the tile that starts here and goes on
};

VSA_DEVICE int tokens_of(const PagedSelectParams& p, int s) { return min(max(__ldg(p.lengths + s), 0), p.width * kBlock); }
VSA_DEVICE int pages_of(const PagedSelectParams& p, int s) { return (tokens_of(p, s) + kBlock - 1) / kBlock; }

VSA_DEVICE void copy16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// kHeads query heads share a pass; 0 = no coarse branch.
template <int kType, int kHeads>
__global__ void __launch_bounds__(kScoreThreads, 1) page_scores_kernel(const __grid_constant__ SelectParams a) {
  constexpr int kG = kHeads > 0 ? kHeads : 1;
  constexpr int kCopies = kHeads > 0 ? 4 : 2;  // 16-byte pieces of a lane per step: two of k_sum, two of v_sum
  extern __shared__ __align__(16) float4 ring[];
  const PagedSelectParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4, part = lane & 15;
  float4* mine = ring + (warp * kSteps * kCopies) * 32 + lane;  // [step][copy][lane]
  pdl_wait();
  pdl_release();
  const int worker = blockIdx.x * kScoreWarps + warp, heads = p.kv_heads * a.chunks;
  WorkSplit split;
  const WorkRange range = find_work([&](int s) { return pages_of(p, s); }, p.requests, heads, worker, a.workers, kLeastUnits, split);
  int s = range.request, hv = range.head, unit = range.unit, left = range.end - range.begin;
  if (kHeads > 0 && lane == 0) a.split[worker] = make_int4(0, 0, 0, 0);

  while (left > 0) {
    const int length = tokens_of(p, s), n = (length + kBlock - 1) / kBlock;
    if (n == 0) {
      ++s;
      continue;
    }
    const int last = min(n, unit + left);
    const int head = hv / a.chunks, first_q = (hv % a.chunks) * a.chunk_heads, columns = min(a.chunk_heads, p.group - first_q);
    const bool scoring = p.chosen != nullptr && n > p.keep && hv % a.chunks == 0;
    if (kHeads > 0 || scoring) {
      const int32_t* table = p.tables + s * p.table_stride;
      // Steps of two pages; the table is looked up 32 pages at a time, one round ahead of the copies.
      const int steps = (last - unit + 1) / 2;
      int page = unit + lane < last ? __ldg(table + unit + lane) : -1, next = -1;
      const auto issue = [&](int step) {
        const int at = 2 * step + half;
        if (step < steps) {
          if (step > 0 && step % 16 == 0) page = next;
          if (step % 16 == 0) next = unit + 2 * step + 32 + lane < last ? __ldg(table + unit + 2 * step + 32 + lane) : -1;
        }
        const int id = __shfl_sync(~0u, page, at % 32);
        const bool valid = step < steps && id >= 0 && id < p.pages;
        if (part == 0 && unit + at < last && step < steps && !valid) paged_error(p.status, kPagedBadPage);
        const long long row = ((valid ? static_cast<long long>(id) : 0) * p.kv_heads + head) * kDim + 4 * part;
        float4* dst = mine + (step % kSteps) * kCopies * 32;
        copy16(dst, p.k_sum + row, valid);
        copy16(dst + 32, p.k_sum + row + 64, valid);
        if (kHeads > 0) {
          copy16(dst + 64, p.v_sum + row, valid);
          copy16(dst + 96, p.v_sum + row + 64, valid);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return valid;
      };
      unsigned live = 0;  // bit step % kSteps: this lane's page of the step exists
#pragma unroll
      for (int i = 0; i < kSteps - 1; ++i) live |= static_cast<unsigned>(issue(i)) << i;

      // This lane's dims: 4 part + 0..3 and 64 more.
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + s * p.q_row_stride + static_cast<long long>(head) * p.group * p.q_head_stride;
      double sum_q[8];
      if (scoring) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum_q[i] = 0.;
        for (int g = 0; g < p.group; ++g) {
          const uint2 x = __ldg(reinterpret_cast<const uint2*>(q + g * p.q_head_stride) + part), y = __ldg(reinterpret_cast<const uint2*>(q + g * p.q_head_stride) + 16 + part);
          const uint32_t w[4] = {x.x, x.y, y.x, y.y};
#pragma unroll
          for (int i = 0; i < 8; ++i) sum_q[i] += unpack1<kType>(static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1))));
        }
      }
      float qf[kG][8], m[kG], l[kG], o[kG][8];
      if (kHeads > 0) {
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          const uint16_t* src = q + static_cast<long long>(first_q + min(g, columns - 1)) * p.q_head_stride;
          const uint2 x = __ldg(reinterpret_cast<const uint2*>(src) + part), y = __ldg(reinterpret_cast<const uint2*>(src) + 16 + part);
          const uint32_t w[4] = {x.x, x.y, y.x, y.y};
          m[g] = -INFINITY, l[g] = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            qf[g][i] = unpack1<kType>(static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)))) * (p.scale * kLog2e);
            o[g][i] = 0.f;
          }
        }
      }
      double* score = scoring ? a.score + (static_cast<long long>(s) * p.kv_heads + head) * p.width : nullptr;
      for (int step = 0; step < steps; ++step) {
        const bool fresh = issue(step + kSteps - 1);
        const int at_new = (step + kSteps - 1) % kSteps, at = step % kSteps;
        asm volatile("cp.async.wait_group %0;" ::"n"(kSteps - 1) : "memory");
        const float4* src = mine + at * kCopies * 32;
        const float4 k0 = src[0], k1 = src[32];
        const int i = unit + 2 * step + half;
        const bool valid = (live >> at) & 1;
        live = (live & ~(1u << at_new)) | (static_cast<unsigned>(fresh) << at_new);
        const float kk[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
        const int tokens = min(kBlock, length - i * kBlock);
        if (scoring) {
          double x = 0.;
#pragma unroll
          for (int d = 0; d < 8; ++d) x = fma(sum_q[d], static_cast<double>(kk[d]), x);
#pragma unroll
          for (int d = 8; d > 0; d /= 2) x += __shfl_xor_sync(~0u, x, d);
          if (part == 0 && i < last) {
            x = tokens == kBlock ? x * (1. / kBlock) : x / static_cast<double>(tokens);
            score[i] = isnan(x) ? kTopScore : fmin(fmax(x, -kTopScore), kTopScore);
          }
        }
        if (kHeads > 0) {
          const float4 v0 = src[64], v1 = src[96];
          const float vv[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
          const float inv = tokens == kBlock ? 1.f / kBlock : 1.f / static_cast<float>(max(tokens, 1));
          float x[kG];
#pragma unroll
          for (int g = 0; g < kG; ++g) {
            x[g] = 0.f;
#pragma unroll
            for (int d = 0; d < 8; ++d) x[g] = fmaf(qf[g][d], kk[d], x[g]);
          }
#pragma unroll
          for (int d = 8; d > 0; d /= 2)
#pragma unroll
            for (int g = 0; g < kG; ++g) x[g] += __shfl_xor_sync(~0u, x[g], d);
#pragma unroll
          for (int g = 0; g < kG; ++g) {
            const float sc = valid ? x[g] * inv : -INFINITY;
            if (sc > m[g]) {
              const float shrink = exp2_fast(m[g] - sc);
              m[g] = sc;
              l[g] *= shrink;
#pragma unroll
              for (int d = 0; d < 8; ++d) o[g][d] *= shrink;
            }
            const float w = valid ? exp2_fast(sc - finite_or_zero(m[g])) : 0.f;
            l[g] += w;
            if (valid) {
#pragma unroll
              for (int d = 0; d < 8; ++d) o[g][d] = fmaf(w * inv, vv[d], o[g][d]);
            }
          }
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      if (kHeads > 0) {
        const bool starts = unit == 0, ends = last == n;
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          const float top = fmaxf(m[g], __shfl_xor_sync(~0u, m[g], 16));
          const float f = exp2_fast(m[g] - finite_or_zero(top));
          float sum = l[g] * f, y[8];
          sum += __shfl_xor_sync(~0u, sum, 16);
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            y[d] = o[g][d] * f;
            y[d] += __shfl_xor_sync(~0u, y[d], 16);
          }
          if (g >= columns) continue;
          float4 out = half == 0 ? make_float4(y[0], y[1], y[2], y[3]) : make_float4(y[4], y[5], y[6], y[7]);
          const int d = 64 * half + 4 * part;
          if (starts && ends) {
            const float f = sum == 0.f ? 0.f : 1.f / sum;
            const long long row = (static_cast<long long>(s) * p.kv_heads + head) * p.group + first_q + g;
            if (sum == 0.f) out = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(p.coarse + row * kDim + d) = make_float4(out.x * f, out.y * f, out.z * f, out.w * f);
          } else {
            const long long slot = (2LL * worker + (starts ? 1 : 0)) * a.chunk_heads + g;
            *reinterpret_cast<float4*>(a.partials + slot * kDim + d) = out;
            if (lane == 0) a.stats[slot] = make_float2(top, sum);
          }
        }
        if (lane == 0 && starts && !ends) a.split[worker] = make_int4(s, hv, split.owner(range.end + (n - last) - 1), 1);
      }
    }
    left -= last - unit;
    unit = 0;
    if (last == n && ++hv == heads) hv = 0, ++s;
  }
  // Requests without tokens have no pages.
  if (kHeads > 0)
    for (int e = worker; e < p.requests; e += a.workers)
      if (pages_of(p, e) == 0)
        for (int i = lane; i < p.kv_heads * p.group * (kDim / 4); i += 32)
          reinterpret_cast<float4*>(p.coarse)[static_cast<long long>(e) * p.kv_heads * p.group * (kDim / 4) + i] = make_float4(0.f, 0.f, 0.f, 0.f);
}

struct ChooseShared {
  int hist[kBins];
  int sums[kChooseWarps];
  double low[kChooseWarps], high[kChooseWarps];
  int border, above;
};

// Inclusive prefix sum over the block and the block's total.
VSA_DEVICE int2 block_scan(int x, int* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int y = __shfl_up_sync(~0u, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kChooseWarps; ++w) {
    const int s = sums[w];
    if (w < warp) before += s;
    all += s;
  }
  return make_int2(x + before, all);
}

// Lowest and highest value over the block.
VSA_DEVICE void block_bounds(double& a, double& b, ChooseShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 16; d > 0; d /= 2) {
    a = fmin(a, __shfl_xor_sync(~0u, a, d));
    b = fmax(b, __shfl_xor_sync(~0u, b, d));
  }
  __syncthreads();
  if (lane == 0) sh.low[warp] = a, sh.high[warp] = b;
  __syncthreads();
  a = sh.low[0], b = sh.high[0];
#pragma unroll
  for (int w = 1; w < kChooseWarps; ++w) a = fmin(a, sh.low[w]), b = fmax(b, sh.high[w]);
}

// One CTA: list the pages to keep, ascending.
__device__ void choose_pages(const PagedSelectParams& p, const double* from, double* score, int n, int32_t* out, ChooseShared& sh) {
  const int tid = threadIdx.x;
  for (int i = min(n, p.keep) + tid; i < p.keep; i += kChooseThreads) out[i] = -1;
  if (n <= p.keep) {
    for (int i = tid; i < n; i += kChooseThreads) out[i] = i;
    return;
  }
  const int begin = p.first, end = n - p.last;  // candidates; the others are always kept
  int need = p.keep - p.first - p.last;
  double low = INFINITY, high = -INFINITY;      // candidates above `high` are in, below `low` out
  for (int i = begin + tid; i < end; i += kChooseThreads) {
    const double s = from[i];
    score[i] = s;
    low = fmin(low, s), high = fmax(high, s);
  }
  block_bounds(low, high, sh);
  int ties = n;  // candidates equal to `low` that are in, lowest first
  if (need == 0) low = INFINITY;
  while (need > 0) {
    if (low == high) {  // all that is left ties
      ties = need;
      break;
    }
    for (int i = tid; i < kBins; i += kChooseThreads) sh.hist[i] = 0;
    __syncthreads();
    const double per = (kBins - 1) / (high - low);
    for (int i = begin + tid; i < end; i += kChooseThreads) {
      const double s = score[i];
      if (s >= low && s <= high) atomicAdd(&sh.hist[min(kBins - 1, static_cast<int>((s - low) * per))], 1);
    }
    __syncthreads();
    // Bins from the top: thread t owns the next few below those of t - 1.
    constexpr int kOwn = kBins / kChooseThreads;
    int own[kOwn], mine = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) mine += own[i] = sh.hist[kBins - 1 - (tid * kOwn + i)];
    int above = block_scan(mine, sh.sums).x - mine;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (above < need && above + own[i] >= need) sh.border = kBins - 1 - (tid * kOwn + i), sh.above = above;
      above += own[i];
    }
    __syncthreads();
    const int border = sh.border, in_border = sh.hist[border];
    need -= sh.above;
    // Narrow the interval to the border bin's own scores.
    double a = INFINITY, b = -INFINITY;
    for (int i = begin + tid; i < end; i += kChooseThreads) {
      const double s = score[i];
      if (s >= low && s <= high && min(kBins - 1, static_cast<int>((s - low) * per)) == border) a = fmin(a, s), b = fmax(b, s);
    }
    block_bounds(a, b, sh);
    low = a, high = b;
    if (need == in_border) break;  // the whole bin is in
  }
  int tied = 0, listed = 0;
  for (int base = 0; base < n; base += kChooseThreads) {
    const int i = base + tid;
    const bool always = i < n && (i < begin || i >= end), candidate = i < n && !always;
    const double s = candidate ? score[i] : 0.;
    const bool tie = candidate && s == low;
    bool in = always || (candidate && s > low) || tie;
    if (ties < n) {  // not all of the ties are in
      const int2 t = block_scan(tie, sh.sums);
      in = in && (!tie || tied + t.x <= ties);
      tied += t.y;
    }
    const int2 c = block_scan(in, sh.sums);
    if (in) out[listed + c.x - 1] = i;
    listed += c.y;
  }
}

// CTAs below `tiles` choose pages, the others join partial results.
__global__ void __launch_bounds__(kChooseThreads) page_choose_kernel(const __grid_constant__ SelectParams a, int tiles) {
  extern __shared__ __align__(16) double score[];  // [width]
  __shared__ ChooseShared sh;
  const PagedSelectParams& p = a.p;
  pdl_wait();
  pdl_release();
  if (static_cast<int>(blockIdx.x) < tiles) {
    const int n = pages_of(p, blockIdx.x / p.kv_heads);
    choose_pages(p, a.score + static_cast<long long>(blockIdx.x) * p.width, score, n, p.chosen + static_cast<long long>(blockIdx.x) * p.keep, sh);
    return;
  }
  // One warp per (worker, query head).
  const int x = (blockIdx.x - tiles) * kChooseWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int first = x / a.chunk_heads, col = x % a.chunk_heads;
  if (first >= a.workers) return;
  const int4 tile = a.split[first];
  if (tile.w == 0) return;
  const int head = tile.y / a.chunks, first_q = (tile.y % a.chunks) * a.chunk_heads;
  if (col >= min(a.chunk_heads, p.group - first_q)) return;
  float top = -INFINITY;
  for (int w = first + lane; w <= tile.z; w += 32) top = fmaxf(top, a.stats[(2LL * w + (w == first ? 1 : 0)) * a.chunk_heads + col].x);
#pragma unroll
  for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  float sum = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int w = first; w <= tile.z; ++w) {
    const long long slot = (2LL * w + (w == first ? 1 : 0)) * a.chunk_heads + col;
    const float2 st = a.stats[slot];
    const float4 v = *reinterpret_cast<const float4*>(a.partials + slot * kDim + 4 * lane);
    const float f = exp2_fast(st.x - finite_or_zero(top));
    sum += f * st.y;
    y.x += f * v.x, y.y += f * v.y, y.z += f * v.z, y.w += f * v.w;
  }
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  if (sum == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
  const long long row = (static_cast<long long>(tile.x) * p.kv_heads + head) * p.group + first_q + col;
  *reinterpret_cast<float4*>(p.coarse + row * kDim + 4 * lane) = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
}

struct Workspace {
  int64_t score, partials, stats, split, bytes;
};
Workspace workspace_of(int64_t requests, int64_t kv_heads, int group, int64_t width, bool choose, bool coarse) {
  const int columns = group < kColumnsMax ? group : kColumnsMax;
  Workspace w{};
  int64_t at = choose ? requests * kv_heads * width * 8 : 0;
  at = (at + 15) / 16 * 16;
  if (coarse) {
    w.split = at, at += kWorkersMax * 16;
    w.partials = at, at += 2LL * kWorkersMax * columns * kDim * 4;
    w.stats = at, at += 2LL * kWorkersMax * columns * 8;
  }
  w.bytes = at > 0 ? at : 16;
  return w;
}

template <int kType, int kHeads>
cudaError_t launch(const SelectParams& a, cudaStream_t stream) {
  const int smem = kScoreWarps * kSteps * (kHeads > 0 ? 4 : 2) * 32 * 16;
  return launch_overlapped(page_scores_kernel<kType, kHeads>, dim3(a.workers / kScoreWarps), kScoreThreads, smem, stream, a);
}
template <int kType>
cudaError_t launch_type(const SelectParams& a, cudaStream_t stream) {
  if (a.p.coarse == nullptr) return launch<kType, 0>(a, stream);
  if (a.chunk_heads == 1) return launch<kType, 1>(a, stream);
  if (a.chunk_heads == 2) return launch<kType, 2>(a, stream);
  return launch<kType, 4>(a, stream);
}

}  // namespace

int64_t paged_select_workspace_bytes(int requests, int kv_heads, int group, int width, bool choose, bool coarse) {
  return workspace_of(requests, kv_heads, group, width, choose, coarse).bytes;
}

cudaError_t launch_paged_select(const PagedSelectParams& p, cudaStream_t stream) {
  SelectParams a{};
  a.p = p;
  const bool choose = p.chosen != nullptr, coarse = p.coarse != nullptr;
  // Without the coarse branch one pass serves the whole group.
  a.chunks = coarse ? (p.group + kColumnsMax - 1) / kColumnsMax : 1;
  a.chunk_heads = (p.group + a.chunks - 1) / a.chunks;
  int device = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (err != cudaSuccess) return err;
  a.workers = (sms * kScoreWarps < kWorkersMax ? sms : kWorkersMax / kScoreWarps) * kScoreWarps;
  const Workspace w = workspace_of(p.requests, p.kv_heads, p.group, p.width, choose, coarse);
  a.score = reinterpret_cast<double*>(p.workspace);
  a.split = reinterpret_cast<int4*>(p.workspace + w.split);
  a.partials = reinterpret_cast<float*>(p.workspace + w.partials);
  a.stats = reinterpret_cast<float2*>(p.workspace + w.stats);
  err = p.dtype == kBf16 ? launch_type<kBf16>(a, stream) : launch_type<kFp16>(a, stream);
  if (err != cudaSuccess) return err;
  const int tiles = choose ? p.requests * p.kv_heads : 0;
  const int joins = coarse ? (a.workers * a.chunk_heads + kChooseWarps - 1) / kChooseWarps : 0;
  return launch_overlapped(page_choose_kernel, dim3(tiles + joins), kChooseThreads, choose ? p.width * 8 : 0, stream, a, tiles);
}

}  // namespace vsa
