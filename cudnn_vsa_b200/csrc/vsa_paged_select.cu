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
// kernel; the 64-bit products ride along.
//
// A cluster of up to eight CTAs shares the pages of one (request, key/value head).  Eight lanes
// take a page (64 bytes of its sum each), so that a warp has four pages in flight.  Scores go to
// the leading CTA's shared memory; it narrows the interval that holds the last score kept with
// histograms of 2048 equal bins over [lowest, highest candidate] - scores of real inputs are spread,
// so the first pass leaves a few candidates - and lists the pages in ascending order.  Coarse
// partial results (running maximum, sum, output) are joined over lanes, warps and CTAs.
#include <cooperative_groups.h>

#include "vsa_paged_common.cuh"

namespace vsa {

namespace {

namespace cg = cooperative_groups;

constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kBins = 2048;
constexpr double kTopScore = 1e200;  // stands for +infinity and NaN: above every finite score
constexpr float kLog2e = 1.4426950408889634f;

VSA_DEVICE float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
VSA_DEVICE float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

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
  for (int w = 0; w < kSelectWarps; ++w) {
    const int s = sums[w];
    if (w < warp) before += s;
    all += s;
  }
  return make_int2(x + before, all);
}

struct SelectShared {
  float o[kSelectWarps][4][kDim];
  float m[kSelectWarps][4], l[kSelectWarps][4];
  float join_o[4][kDim], join_m[4], join_l[4];
  int hist[kBins];
  int sums[kSelectWarps];
  double low[kSelectWarps], high[kSelectWarps];
  int border, above;
};

// The leading CTA: list the pages to keep, ascending.
__device__ void choose_pages(const PagedSelectParams& p, const double* score, int n, int32_t* out, SelectShared& sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = min(n, p.keep) + tid; i < p.keep; i += kSelectThreads) out[i] = -1;
  if (n <= p.keep) {
    for (int i = tid; i < n; i += kSelectThreads) out[i] = i;
    return;
  }
  const int begin = p.first, end = n - p.last;  // candidates; the others are always kept
  int need = p.keep - p.first - p.last;
  double low = -INFINITY, high = INFINITY;      // candidates above `high` are in, below `low` out
  int ties = n;                                 // candidates equal to `low` that are in, lowest first
  if (need == 0) low = INFINITY;
  while (need > 0) {
    // The candidates' own lowest and highest score.
    double a = INFINITY, b = -INFINITY;
    for (int i = begin + tid; i < end; i += kSelectThreads) {
      const double s = score[i];
      if (s >= low && s <= high) a = fmin(a, s), b = fmax(b, s);
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
      a = fmin(a, __shfl_xor_sync(~0u, a, d));
      b = fmax(b, __shfl_xor_sync(~0u, b, d));
    }
    __syncthreads();
    if (lane == 0) sh.low[warp] = a, sh.high[warp] = b;
    for (int i = tid; i < kBins; i += kSelectThreads) sh.hist[i] = 0;
    __syncthreads();
    low = sh.low[0], high = sh.high[0];
#pragma unroll
    for (int w = 1; w < kSelectWarps; ++w) low = fmin(low, sh.low[w]), high = fmax(high, sh.high[w]);
    if (low == high) {  // all that is left ties
      ties = need;
      break;
    }
    const double per = (kBins - 1) / (high - low);
    for (int i = begin + tid; i < end; i += kSelectThreads) {
      const double s = score[i];
      if (s >= low && s <= high) atomicAdd(&sh.hist[min(kBins - 1, static_cast<int>((s - low) * per))], 1);
    }
    __syncthreads();
    // Bins from the top: thread t owns the eight bins below kBins - 8 t.
    constexpr int kOwn = kBins / kSelectThreads;
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
    a = INFINITY, b = -INFINITY;
    for (int i = begin + tid; i < end; i += kSelectThreads) {
      const double s = score[i];
      if (s >= low && s <= high && min(kBins - 1, static_cast<int>((s - low) * per)) == border) a = fmin(a, s), b = fmax(b, s);
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
      a = fmin(a, __shfl_xor_sync(~0u, a, d));
      b = fmax(b, __shfl_xor_sync(~0u, b, d));
    }
    __syncthreads();
    if (lane == 0) sh.low[warp] = a, sh.high[warp] = b;
    __syncthreads();
    low = sh.low[0], high = sh.high[0];
#pragma unroll
    for (int w = 1; w < kSelectWarps; ++w) low = fmin(low, sh.low[w]), high = fmax(high, sh.high[w]);
    if (need == in_border) break;  // the whole bin is in
  }
  int tied = 0, listed = 0;
  for (int base = 0; base < n; base += kSelectThreads) {
    const int i = base + tid;
    const bool always = i < n && (i < begin || i >= end), candidate = i < n && !always;
    const double s = candidate ? score[i] : 0.;
    const bool tie = candidate && s == low;
    const int2 t = block_scan(tie, sh.sums);
    const bool in = always || (candidate && s > low) || (tie && tied + t.x <= ties);
    const int2 c = block_scan(in, sh.sums);
    if (in) out[listed + c.x - 1] = i;
    tied += t.y;
    listed += c.y;
  }
}

// kHeads query heads share one pass over the pages' sums; 0 = no coarse branch.
template <int kType, int kHeads>
__global__ void __launch_bounds__(kSelectThreads) paged_select_kernel(PagedSelectParams p) {
  extern __shared__ __align__(16) double score[];  // [width], the leading CTA's is used
  __shared__ __align__(16) SelectShared sh;
  constexpr int kG = kHeads > 0 ? kHeads : 1;
  __shared__ __align__(16) float qs[kG][kDim];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), size = static_cast<int>(cluster.num_blocks());
  const int request = blockIdx.z, head = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, part = lane & 7;
  const int length = min(max(p.lengths[request], 0), p.width * kBlock);
  const int n = (length + kBlock - 1) / kBlock;
  const int begin = static_cast<int>(static_cast<long long>(n) * rank / size);
  const int end = static_cast<int>(static_cast<long long>(n) * (rank + 1) / size);
  const bool scoring = p.chosen != nullptr && n > p.keep;
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + request * p.q_row_stride + static_cast<long long>(head) * p.group * p.q_head_stride;
  double* lead = cluster.map_shared_rank(score, 0);

  // The group's summed query, 16 dims per lane: dims 4 * (part + 8 i) + 0..3.
  double qsum[16];
  if (scoring) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = 4 * (part + 8 * (i / 4)) + i % 4;
      double sum = 0.;
      for (int g = 0; g < p.group; ++g) sum += unpack1<kType>(q[g * p.q_head_stride + d]);
      qsum[i] = sum;
    }
  }
  cluster.sync();  // the leading CTA runs before its shared memory is written
  const int32_t* table = p.tables + request * p.table_stride;
  const int rounds = kHeads > 0 ? (p.group + kG - 1) / kG : 1;
  for (int round = 0; round < rounds; ++round) {
    const int heads = min(kG, p.group - round * kG);
    if (kHeads > 0) {
      __syncthreads();
      for (int i = tid; i < kG * kDim; i += kSelectThreads)
        qs[i / kDim][i % kDim] = i / kDim < heads ? unpack1<kType>(q[(round * kG + i / kDim) * p.q_head_stride + i % kDim]) * (p.scale * kLog2e) : 0.f;
      __syncthreads();
    }
    float m[kG], l[kG], o[kG][16];
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      m[g] = -INFINITY, l[g] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) o[g][i] = 0.f;
    }
    const bool score_now = scoring && round == 0;
    if (kHeads > 0 || score_now) {
      for (int base = begin + warp * 4; base < end; base += kSelectWarps * 4) {
        const int i = base + lane / 8;
        int page = i < end ? table[i] : -1;
        if (i < end && (page < 0 || page >= p.pages)) {
          paged_error(p.status, kPagedBadPage);
          page = -1;
        }
        const float tokens = static_cast<float>(min(kBlock, length - i * kBlock));
        float4 k[4], v[4];
        const long long row = (static_cast<long long>(max(page, 0)) * p.kv_heads + head) * (kDim / 4) + part;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          k[c] = page >= 0 ? __ldg(reinterpret_cast<const float4*>(p.k_sum) + row + 8 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
          if (kHeads > 0) v[c] = page >= 0 ? __ldg(reinterpret_cast<const float4*>(p.v_sum) + row + 8 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (score_now) {
          double s = 0.;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s = fma(qsum[4 * c], static_cast<double>(k[c].x), s);
            s = fma(qsum[4 * c + 1], static_cast<double>(k[c].y), s);
            s = fma(qsum[4 * c + 2], static_cast<double>(k[c].z), s);
            s = fma(qsum[4 * c + 3], static_cast<double>(k[c].w), s);
          }
#pragma unroll
          for (int d = 4; d > 0; d /= 2) s += __shfl_xor_sync(~0u, s, d);
          s /= static_cast<double>(tokens);
          if (part == 0 && i < end) lead[i] = isnan(s) ? kTopScore : fmin(fmax(s, -kTopScore), kTopScore);
        }
        if (kHeads > 0) {
          const float inv = 1.f / tokens;
#pragma unroll
          for (int g = 0; g < kG; ++g) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float4 x = reinterpret_cast<const float4*>(qs[g])[part + 8 * c];
              s += x.x * k[c].x + x.y * k[c].y + x.z * k[c].z + x.w * k[c].w;
            }
#pragma unroll
            for (int d = 4; d > 0; d /= 2) s += __shfl_xor_sync(~0u, s, d);
            s *= inv;
            if (page < 0) continue;
            if (s > m[g]) {
              const float shrink = exp2_fast(m[g] - s);
              m[g] = s;
              l[g] *= shrink;
#pragma unroll
              for (int d = 0; d < 16; ++d) o[g][d] *= shrink;
            }
            const float w = exp2_fast(s - finite_or_zero(m[g]));
            l[g] += w;
            const float wv = w * inv;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              o[g][4 * c] += wv * v[c].x, o[g][4 * c + 1] += wv * v[c].y;
              o[g][4 * c + 2] += wv * v[c].z, o[g][4 * c + 3] += wv * v[c].w;
            }
          }
        }
      }
    }
    if (kHeads > 0) {
      // Four page groups of the warp, then the warps, then the CTAs.
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        float top = fmaxf(m[g], __shfl_xor_sync(~0u, m[g], 8));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
        const float w = exp2_fast(m[g] - finite_or_zero(top));
        l[g] *= w;
        l[g] += __shfl_xor_sync(~0u, l[g], 8);
        l[g] += __shfl_xor_sync(~0u, l[g], 16);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x = o[g][i] * w;
          x += __shfl_xor_sync(~0u, x, 8);
          x += __shfl_xor_sync(~0u, x, 16);
          if (lane < 8) sh.o[warp][g][4 * (part + 8 * (i / 4)) + i % 4] = x;
        }
        if (lane == 0) sh.m[warp][g] = top, sh.l[warp][g] = l[g];
      }
      __syncthreads();
      for (int x = tid; x < kG * kDim; x += kSelectThreads) {
        const int g = x / kDim, d = x % kDim;
        float top = -INFINITY, sum = 0.f, all = 0.f;
#pragma unroll
        for (int w = 0; w < kSelectWarps; ++w) top = fmaxf(top, sh.m[w][g]);
#pragma unroll
        for (int w = 0; w < kSelectWarps; ++w) {
          const float f = exp2_fast(sh.m[w][g] - finite_or_zero(top));
          sum += f * sh.o[w][g][d];
          all += f * sh.l[w][g];
        }
        sh.join_o[g][d] = sum;
        if (d == 0) sh.join_m[g] = top, sh.join_l[g] = all;
      }
      cluster.sync();
      // Spread over the CTAs: element x of the round's outputs belongs to CTA x / 128 % size.
      for (int x = tid; x < heads * kDim; x += kSelectThreads) {
        const int g = x / kDim, d = x % kDim;
        if (g % size != rank) continue;
        float top = -INFINITY, sum = 0.f, all = 0.f;
        for (int c = 0; c < size; ++c) top = fmaxf(top, *cluster.map_shared_rank(&sh.join_m[g], c));
        for (int c = 0; c < size; ++c) {
          const float f = exp2_fast(*cluster.map_shared_rank(&sh.join_m[g], c) - finite_or_zero(top));
          sum += f * *cluster.map_shared_rank(&sh.join_o[g][d], c);
          all += f * *cluster.map_shared_rank(&sh.join_l[g], c);
        }
        const long long row = (static_cast<long long>(request) * p.kv_heads + head) * p.group + round * kG + g;
        p.coarse[row * kDim + d] = all == 0.f ? 0.f : sum / all;
      }
    }
    // Orders the scores before the choice, and the partial results' readers before the next round.
    cluster.sync();
  }
  if (rank == 0 && p.chosen != nullptr)
    choose_pages(p, score, n, p.chosen + (static_cast<long long>(request) * p.kv_heads + head) * p.keep, sh);
}

template <int kType, int kHeads>
cudaError_t launch(const PagedSelectParams& p, int size, cudaStream_t stream) {
  auto* kernel = paged_select_kernel<kType, kHeads>;
  const int smem = p.chosen != nullptr ? p.width * static_cast<int>(sizeof(double)) : 0;
  if (smem > 16 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return err;
  }
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(size, p.kv_heads, p.requests);
  config.blockDim = dim3(kSelectThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = size, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, p);
}

template <int kType>
cudaError_t launch_type(const PagedSelectParams& p, int size, cudaStream_t stream) {
  if (p.coarse == nullptr) return launch<kType, 0>(p, size, stream);
  if (p.group == 1) return launch<kType, 1>(p, size, stream);
  if (p.group == 2) return launch<kType, 2>(p, size, stream);
  return launch<kType, 4>(p, size, stream);
}

}  // namespace

cudaError_t launch_paged_select(const PagedSelectParams& p, cudaStream_t stream) {
  // As many CTAs to a (request, head) as fill the device, but no fewer than 32 pages for each.
  const long long tiles = static_cast<long long>(p.requests) * p.kv_heads;
  int size = 1;
  while (size < 8 && tiles * size < 2 * 148 && p.width >= 64 * size) size *= 2;
  return p.dtype == kBf16 ? launch_type<kBf16>(p, size, stream) : launch_type<kFp16>(p, size, stream);
}

}  // namespace vsa
