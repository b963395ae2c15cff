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
//                       It takes 16 pages a round, fetched by cp.async into buffers of its own (17 KiB
//                       a warp, twelve warps to an SM): the next keys fly while the values are used
//                       and the other way round.  Two lanes score a page (rows are 528 bytes apart, so
//                       that the lanes' 16-byte reads meet all banks): hardly any sums across lanes,
//                       and a query value read once serves 16 pages.  For the values a lane holds
//                       four dims.  Incomplete tiles go to the workspace.  16 requests of 1,776 pages, 12
//                       heads, 347 MB: 58 us, of which HBM needs 53; without the coarse branch, 174 MB in
//                       36 us, the conversions to 64 bits take as long as the loads.
//   page_choose_kernel  Joins the incomplete tiles and chooses the pages, one CTA per
//                       (request, head): a histogram of 2048 equal bins over [lowest, highest] FP32
//                       rounding of the candidates' scores (rounding keeps their order) finds the bin that
//                       holds the last page kept; its few candidates are ranked by their 64-bit scores.
//                       A bin with more than 256 candidates is narrowed in 64 bits first.  The pages
//                       are listed in ascending order from a bit map.  1,776 pages: about 5 us.
//   page_short_kernel   Short requests (tables of up to 128 pages): one CTA per (request, head) does
//                       it all, a launch less and many chains of steps side by side.  CTAs of 256, 128 or 64
//                       threads, so that the SMs hold all tiles (512 threads each): 128 / 512 / 2,048 tiles of
//                       16 pages, four heads a group, with the coarse branch, take 7.4 / 15.0 / 57 us with 256
//                       threads, 7.4 / 8.6 / 34 us with 128, 9.1 / 9.8 / 24 us with 64 and 13.8 / 19.2 / 42 us in
//                       two kernels; 128 tiles of 64 pages 9.0, 11.7, 18.8 and 17.6 us.  With 128 pages and the
//                       coarse branch the two kernels win above 592 tiles (2,048: 95 against 85 us; 512: 28
//                       against 28 us), without it never (39 against 45 us).
#include "vsa_paged_common.cuh"

namespace vsa {

namespace {

constexpr int kWorkersMax = 160 * 20;
constexpr int kRound = 16;                // pages of a round, two lanes each
constexpr int kRowFloats = kDim + 4;      // of a buffered row
// Pages a worker takes at least: few workers leave few results to join, many take less than a round each.  24 tiles of
// 400 pages, five heads a group: 18.6, 14.3, 14.3 us with 4, 8, 16; six tiles of 150 pages 14.5, 15.5, 16.4.
constexpr int kLeastUnits = 8;
constexpr int kColumnsMax = 8;            // query heads that share one pass over the sums
constexpr int kChooseThreads = 256, kChooseWarps = kChooseThreads / 32;
constexpr int kShortPages = 128;
constexpr double kTopScore = 1e200;  // stands for +infinity and NaN: above every score of finite inputs

struct SelectParams {
  PagedSelectParams p;
  int chunks, chunk_heads;  // a group is taken in `chunks` parts of up to `chunk_heads` query heads
  int workers;
  double* score;            // [requests, kv_heads, width]
  float* partials;          // [2 * workers][chunk_heads][128]
  float2* stats;            // [2 * workers][chunk_heads]
};

VSA_DEVICE double finite_score(double x) { return isnan(x) ? kTopScore : fmin(fmax(x, -kTopScore), kTopScore); }
VSA_DEVICE int tokens_of(const PagedSelectParams& p, int s) { return min(max(p.lengths[s], 0), p.width * kBlock); }
VSA_DEVICE int pages_of(const PagedSelectParams& p, int s) { return (tokens_of(p, s) + kBlock - 1) / kBlock; }

VSA_DEVICE void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
template <int kPending>
VSA_DEVICE void copies_done() {  // all but the last kPending groups of this warp's lanes
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
  __syncwarp();
}

template <int kG, bool kCoarse>
struct alignas(16) ScoreShared {  // of one warp
  // As many warps as the shared memory holds.
  static constexpr int kWarps = !kCoarse ? 20 : kG <= 2 ? 12 : kG <= 4 ? 11 : kG <= 6 ? 10 : 9;
  float k[kRound][kRowFloats];
  float v[kCoarse ? kRound : 1][kRowFloats];
  double sum_q[kDim];
  float q[kG][kDim];
  f32x2 p[kG][kRound];  // probabilities, twice each
};

// kHeads query heads share a pass; 0 = no coarse branch.
template <int kType, int kHeads>
__global__ void __launch_bounds__(32 * ScoreShared<(kHeads > 0 ? kHeads : 1), (kHeads > 0)>::kWarps, 1)
    page_scores_kernel(const __grid_constant__ SelectParams a) {
  constexpr int kG = kHeads > 0 ? kHeads : 1;
  constexpr bool kCoarse = kHeads > 0;
  using Shared = ScoreShared<kG, kCoarse>;
  extern __shared__ __align__(16) uint8_t raw[];
  const PagedSelectParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, own = lane & 15, half = lane >> 4;
  Shared& sh = reinterpret_cast<Shared*>(raw)[warp];
  if (!p.early) {
    pdl_wait();
    pdl_release();
  }
  const int worker = blockIdx.x * Shared::kWarps + warp, heads = p.kv_heads * a.chunks;
  WorkSplit split;
  const WorkRange range = find_work([&](int s) { return pages_of(p, s); }, p.requests, heads, worker, a.workers, kLeastUnits, split);
  int s = range.request, hv = range.head, unit = range.unit, left = range.end - range.begin;
  bool waited = !p.early;
  const auto wait_once = [&] {
    if (!waited) {
      pdl_wait();
      pdl_release();
      waited = true;
    }
  };
  if (left <= 0) wait_once();

  while (left > 0) {
    const int length = tokens_of(p, s), n = (length + kBlock - 1) / kBlock;
    if (n == 0) {
      ++s;
      continue;
    }
    const int last = min(n, unit + left);
    const int head = hv / a.chunks, first_q = (hv % a.chunks) * a.chunk_heads, columns = min(a.chunk_heads, p.group - first_q);
    const bool scoring = p.chosen != nullptr && n > p.keep && hv % a.chunks == 0;
    if (kCoarse || scoring) {
      const int32_t* table = p.tables + s * p.table_stride;
      // This lane's page of the round that begins at `at`: its row of the sums, or -1.
      const auto look_up = [&](int at) {
        if (at + own >= last) return -1;
        const int page = table[at + own];
        if (page < 0 || page >= p.pages) {
          paged_error(p.status, kPagedBadPage);
          return -1;
        }
        return page * p.kv_heads + head;
      };
      // Eight lanes copy 128 bytes of a row: this lane's rows are 4 i + lane / 8.  What a table leaves
      // out counts as zeros; rows behind `count` are not touched.
      const auto fetch = [&](float* rows, const float* from, int row, int count) {
        const uint32_t dst = smem_u32(rows) + (lane / 8) * kRowFloats * 4 + (lane % 8) * 16;
#pragma unroll
        for (int i = 0; i < kRound / 4; ++i) {
          const int r = __shfl_sync(~0u, row, 4 * i + lane / 8);
          if (4 * i + lane / 8 >= count) continue;
          const float* src = from + static_cast<long long>(max(r, 0)) * kDim + (lane % 8) * 4;
#pragma unroll
          for (int c = 0; c < 4; ++c) copy16(dst + 4 * i * kRowFloats * 4 + c * 128, src + 32 * c, r >= 0);
        }
      };
      const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
      int row = look_up(unit), next = look_up(unit + kRound);
      // The queries, in flight with the table: dims 4 lane .. 4 lane + 3 of the pass's heads.
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + s * p.q_row_stride + static_cast<long long>(head) * p.group * p.q_head_stride;
      const auto load_q = [&](int g) { return reinterpret_cast<const uint2*>(q + static_cast<long long>(g) * p.q_head_stride)[lane]; };
      uint2 qx[kG];
#pragma unroll
      for (int g = 0; g < kG; ++g) qx[g] = load_q(first_q + min(g, columns - 1));
      wait_once();
      fetch(&sh.k[0][0], p.k_sum, row, min(kRound, last - unit));
      commit();
      if (kCoarse) {
        fetch(&sh.v[0][0], p.v_sum, row, min(kRound, last - unit));
        commit();
      }
      if (scoring) {
        double sum[4] = {};
        const auto add = [&](uint2 x) {
          sum[0] += unpack1<kType>(x.x & 0xFFFF), sum[1] += unpack1<kType>(x.x >> 16);
          sum[2] += unpack1<kType>(x.y & 0xFFFF), sum[3] += unpack1<kType>(x.y >> 16);
        };
        if (columns == p.group && columns <= kG) {
#pragma unroll
          for (int g = 0; g < kG; ++g)
            if (g < columns) add(qx[g]);
        } else {
#pragma unroll 4
          for (int g = 0; g < p.group; ++g) add(load_q(g));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sh.sum_q[4 * lane + i] = sum[i];
      }
      float m[kG], l[kG];
      f32x2 o[kG][2];  // dims 4 lane .. 4 lane + 3
      if (kCoarse) {
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          const uint2 x = qx[g];
          const float f = p.scale * kLog2e;
          *reinterpret_cast<float4*>(&sh.q[g][4 * lane]) = make_float4(unpack1<kType>(x.x & 0xFFFF) * f, unpack1<kType>(x.x >> 16) * f,
                                                                       unpack1<kType>(x.y & 0xFFFF) * f, unpack1<kType>(x.y >> 16) * f);
          m[g] = -INFINITY, l[g] = 0.f, o[g][0] = o[g][1] = 0;
        }
      }
      __syncwarp();
      double* score = scoring ? a.score + (static_cast<long long>(s) * p.kv_heads + head) * p.width : nullptr;
      for (int at = unit; at < last; at += kRound) {
        const int count = min(kRound, last - at), i = at + own;
        const int tokens = max(min(kBlock, length - i * kBlock), 1);
        copies_done<kCoarse ? 1 : 0>();  // the keys; the values may still fly
        const float* k_row = sh.k[own] + 64 * half;  // this lane's half of the page's dims
        f32x2 x[kG][2];
        double y[4] = {};
#pragma unroll
        for (int g = 0; g < kG; ++g) x[g][0] = x[g][1] = 0;
        const auto products = [&](bool score_too) {
#pragma unroll 4
          for (int d = 0; d < kDim / 2; d += 4) {
            const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(k_row + d);
            if (score_too) {
              const double2 a0 = *reinterpret_cast<const double2*>(sh.sum_q + 64 * half + d);
              const double2 a1 = *reinterpret_cast<const double2*>(sh.sum_q + 64 * half + d + 2);
              float k0, k1, k2, k3;
              unpack_f32x2(k.x, k0, k1);
              unpack_f32x2(k.y, k2, k3);
              y[0] = fma(a0.x, static_cast<double>(k0), y[0]);
              y[1] = fma(a0.y, static_cast<double>(k1), y[1]);
              y[2] = fma(a1.x, static_cast<double>(k2), y[2]);
              y[3] = fma(a1.y, static_cast<double>(k3), y[3]);
            }
            if (kCoarse) {
#pragma unroll
              for (int g = 0; g < kG; ++g) {
                const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(&sh.q[g][64 * half + d]);
                x[g][0] = fma_f32x2(w.x, k.x, x[g][0]);
                x[g][1] = fma_f32x2(w.y, k.y, x[g][1]);
              }
            }
          }
        };
        if (scoring) products(true);
        else if (kCoarse) products(false);
        __syncwarp();  // all lanes have read the keys
        const int ahead = min(kRound, last - at - kRound);  // pages of the next round
        const bool valid = row >= 0;
        row = next;
        if (ahead > 0) {
          next = look_up(at + 2 * kRound);
          fetch(&sh.k[0][0], p.k_sum, row, ahead);
        }
        commit();
        if (scoring) {
          double sum = (y[0] + y[1]) + (y[2] + y[3]);
          sum += __shfl_xor_sync(~0u, sum, 16);
          sum = tokens == kBlock ? sum * (1. / kBlock) : sum / static_cast<double>(tokens);
          if (half == 0 && i < last) score[i] = finite_score(sum);
        }
        if (kCoarse) {
          const float inv = tokens == kBlock ? 1.f / kBlock : 1.f / static_cast<float>(tokens);
#pragma unroll
          for (int g = 0; g < kG; ++g) {
            float lo, hi;
            unpack_f32x2(add_f32x2(x[g][0], x[g][1]), lo, hi);
            lo += hi;
            lo += __shfl_xor_sync(~0u, lo, 16);
            const float sc = valid ? lo * inv : -INFINITY;
            float top = sc;
#pragma unroll
            for (int d = 8; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
            if (top > m[g]) {  // the same for all lanes
              const float shrink = exp2_fast(m[g] - top);
              m[g] = top;
              l[g] *= shrink;
              const f32x2 both = pack_f32x2(shrink, shrink);
              o[g][0] = mul_f32x2(o[g][0], both), o[g][1] = mul_f32x2(o[g][1], both);
            }
            const float w = valid ? exp2_fast(sc - finite_or_zero(m[g])) : 0.f;
            if (half == 0) {
              l[g] += w;
              sh.p[g][own] = pack_f32x2(w * inv, w * inv);
            }
          }
          copies_done<1>();  // the values; the next keys may still fly
          const auto add_page = [&](int j) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sh.v[j][4 * lane]);
#pragma unroll
            for (int g = 0; g < kG; ++g) {
              const f32x2 w = sh.p[g][j];
              o[g][0] = fma_f32x2(w, v.x, o[g][0]), o[g][1] = fma_f32x2(w, v.y, o[g][1]);
            }
          };
          if (count == kRound) {
#pragma unroll 8
            for (int j = 0; j < kRound; ++j) add_page(j);
          } else {
            for (int j = 0; j < count; ++j) add_page(j);
          }
          __syncwarp();  // all lanes have read the values and probabilities
          if (ahead > 0) fetch(&sh.v[0][0], p.v_sum, row, ahead);
          commit();
        }
      }
      copies_done<0>();
      if (kCoarse) {
        const bool starts = unit == 0, ends = last == n;
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          float sum = l[g];
#pragma unroll
          for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
          if (g >= columns) continue;
          float4 out;
          unpack_f32x2(o[g][0], out.x, out.y);
          unpack_f32x2(o[g][1], out.z, out.w);
          if (starts && ends) {
            const float f = sum == 0.f ? 0.f : 1.f / sum;
            const long long at = (static_cast<long long>(s) * p.kv_heads + head) * p.group + first_q + g;
            if (sum == 0.f) out = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(p.coarse + at * kDim + 4 * lane) = make_float4(out.x * f, out.y * f, out.z * f, out.w * f);
          } else {
            const long long slot = (2LL * worker + (starts ? 1 : 0)) * a.chunk_heads + g;
            *reinterpret_cast<float4*>(a.partials + slot * kDim + 4 * lane) = out;
            if (lane == 0) a.stats[slot] = make_float2(m[g], sum);
          }
        }
      }
    }
    left -= last - unit;
    unit = 0;
    if (last == n && ++hv == heads) hv = 0, ++s;
  }
  wait_once();
  // Requests without tokens have no pages.
  if (kCoarse)
    for (int e = worker; e < p.requests; e += a.workers)
      if (pages_of(p, e) == 0)
        for (long long i = lane; i < static_cast<long long>(p.kv_heads) * p.group * (kDim / 4); i += 32)
          reinterpret_cast<float4*>(p.coarse)[static_cast<long long>(e) * p.kv_heads * p.group * (kDim / 4) + i] = make_float4(0.f, 0.f, 0.f, 0.f);
}

// `kThreads` choose the pages of a request with at most `kMost`, by histograms of `kBins` bins.
template <int kThreads_, int kMost, int kBins_>
struct ChooseShared {
  static constexpr int kThreads = kThreads_, kWarps = kThreads / 32, kBins = kBins_;
  int hist[kBins];
  unsigned map[kMost / 32 + 1];  // pages that are in
  int candidate[kThreads];
  double exact[kThreads];
  int sums[kWarps];
  int low[kWarps], high[kWarps];
  double low64[kWarps], high64[kWarps];
  int border, above, candidates;
};

// Inclusive prefix sum over the block and the block's total.
template <int kWarps>
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
  for (int w = 0; w < kWarps; ++w) {
    const int s = sums[w];
    if (w < warp) before += s;
    all += s;
  }
  return make_int2(x + before, all);
}

// The bin, counted from the top, that holds the `need`-th candidate: sets sh.border and sh.above,
// the candidates in higher bins.
template <class Shared>
VSA_DEVICE void find_border(int need, Shared& sh) {
  constexpr int kBins = Shared::kBins, kOwn = kBins / Shared::kThreads;
  int own[kOwn], mine = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) mine += own[i] = sh.hist[kBins - 1 - (threadIdx.x * kOwn + i)];
  int above = block_scan<Shared::kWarps>(mine, sh.sums).x - mine;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    if (above < need && above + own[i] >= need) sh.border = kBins - 1 - (threadIdx.x * kOwn + i), sh.above = above;
    above += own[i];
  }
  __syncthreads();
}

// Order-preserving integers of FP32 values.
VSA_DEVICE int ordered(float x) {
  const int b = __float_as_int(x);
  return b ^ ((b >> 31) & 0x7fffffff);
}
VSA_DEVICE float unordered(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// One CTA: list the pages to keep, ascending.
template <class Shared>
__device__ void choose_pages(const PagedSelectParams& p, const double* score, float* rounded, int n, int32_t* out, Shared& sh) {
  constexpr int kThreads = Shared::kThreads, kWarps = Shared::kWarps, kBins = Shared::kBins;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = min(n, p.keep) + tid; i < p.keep; i += kThreads) out[i] = -1;
  if (n <= p.keep) {
    for (int i = tid; i < n; i += kThreads) out[i] = i;
    return;
  }
  const int begin = p.first, end = n - p.last;  // candidates; the others are always kept
  int need = p.keep - p.first - p.last;
  int low = 0x7fffffff, high = -0x7fffffff - 1;
  for (int base = begin + tid; base < end; base += 8 * kThreads) {
    double s[8];  // in flight together
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = base + j * kThreads < end ? score[base + j * kThreads] : 0.;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (base + j * kThreads >= end) break;
      const float f = __double2float_rn(fmin(fmax(s[j], -3e38), 3e38));  // keeps the order
      rounded[base + j * kThreads] = f;
      low = min(low, ordered(f)), high = max(high, ordered(f));
    }
  }
  for (int i = tid; i < kBins; i += kThreads) sh.hist[i] = 0;
  low = __reduce_min_sync(~0u, low), high = __reduce_max_sync(~0u, high);
  if (lane == 0) sh.low[warp] = low, sh.high[warp] = high;
  if (tid == 0) sh.candidates = 0;
  __syncthreads();
  low = __reduce_min_sync(~0u, sh.low[lane % kWarps]), high = __reduce_max_sync(~0u, sh.high[lane % kWarps]);
  // Halved, so that the difference of the largest numbers does not overflow; a difference whose
  // reciprocal would is made one bin.
  const float floor_ = 0.5f * unordered(low), span = 0.5f * unordered(high) - floor_;
  const float per = span > 1e-34f ? (kBins - 1) / span : 0.f;
  const auto bin_of = [&](float f) { return min(kBins - 1, static_cast<int>((0.5f * f - floor_) * per)); };
  for (int i = begin + tid; i < end; i += kThreads) atomicAdd(&sh.hist[bin_of(rounded[i])], 1);
  __syncthreads();
  int border = kBins;
  if (need > 0) {
    find_border(need, sh);
    border = sh.border;
    need -= sh.above;
  }
  // A bit for every page above the border; the border's own pages are gathered.
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + tid;
    const bool candidate = i >= begin && i < end;
    const int bin = candidate ? bin_of(rounded[i]) : 0;
    const unsigned in = __ballot_sync(~0u, i < n && (!candidate || bin > border));
    if (lane == 0 && i < n) sh.map[i / 32] = in;
    if (candidate && bin == border) {
      const int slot = atomicAdd(&sh.candidates, 1);
      if (slot < kThreads) sh.candidate[slot] = i;
    }
  }
  __syncthreads();
  if (need > 0 && sh.candidates <= kThreads) {
    // Rank them by 64-bit score; equal scores by page.
    const int count = sh.candidates;
    double mine = 0.;
    if (tid < count) sh.exact[tid] = mine = score[sh.candidate[tid]];
    __syncthreads();
    if (tid < count) {
      const int page = sh.candidate[tid];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += sh.exact[j] > mine || (sh.exact[j] == mine && sh.candidate[j] < page);
      if (rank < need) atomicOr(&sh.map[page / 32], 1u << (page % 32));
    }
  } else if (need > 0) {
    // Many candidates: narrow their interval [low64, high64] in 64 bits until all of it is in or ties.
    const auto candidate = [&](int i) { return bin_of(rounded[i]) == border; };
    double low64 = -INFINITY, high64 = INFINITY;
    const auto narrow = [&](auto&& test) {
      double a = INFINITY, b = -INFINITY;
      for (int i = begin + tid; i < end; i += kThreads)
        if (candidate(i) && score[i] >= low64 && score[i] <= high64 && test(score[i])) a = fmin(a, score[i]), b = fmax(b, score[i]);
#pragma unroll
      for (int d = 16; d > 0; d /= 2) a = fmin(a, __shfl_xor_sync(~0u, a, d)), b = fmax(b, __shfl_xor_sync(~0u, b, d));
      __syncthreads();
      if (lane == 0) sh.low64[warp] = a, sh.high64[warp] = b;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w) a = fmin(a, sh.low64[w]), b = fmax(b, sh.high64[w]);
      low64 = a, high64 = b;
    };
    narrow([](double) { return true; });
    bool all = false;  // every score of the interval is in
    while (!all && low64 < high64) {
      for (int i = tid; i < kBins; i += kThreads) sh.hist[i] = 0;
      __syncthreads();
      const double per64 = (kBins - 1) / (high64 - low64), from = low64;
      const auto bin64 = [&](double s) { return min(kBins - 1, static_cast<int>((s - from) * per64)); };
      for (int i = begin + tid; i < end; i += kThreads)
        if (candidate(i) && score[i] >= low64 && score[i] <= high64) atomicAdd(&sh.hist[bin64(score[i])], 1);
      __syncthreads();
      find_border(need, sh);
      const int at = sh.border;
      need -= sh.above;
      all = need == sh.hist[at];
      narrow([&](double s) { return bin64(s) == at; });
    }
    // Above the interval: in.  Inside it: in, or the lowest pages of those that tie.
    const int each = (n + kThreads - 1) / kThreads, from_page = max(min(tid * each, n), begin), to_page = min(min(tid * each, n) + each, end);
    int mine = 0;
    for (int i = from_page; i < to_page; ++i) mine += candidate(i) && score[i] >= low64 && score[i] <= high64;
    int left = all ? n : need - (block_scan<kWarps>(mine, sh.sums).x - mine);
    for (int i = from_page; i < to_page; ++i)
      if (candidate(i) && (score[i] > high64 || (score[i] >= low64 && score[i] <= high64 && left-- > 0))) atomicOr(&sh.map[i / 32], 1u << (i % 32));
  }
  __syncthreads();
  const int words = (n + 31) / 32;
  int listed = 0;
  for (int base = 0; base < words; base += kThreads) {
    unsigned bits = base + tid < words ? sh.map[base + tid] : 0;
    const int2 c = block_scan<kWarps>(__popc(bits), sh.sums);
    int at = listed + c.x - __popc(bits);
    listed += c.y;
    for (; bits != 0; bits &= bits - 1) out[at++] = 32 * (base + tid) + __ffs(bits) - 1;
  }
}

constexpr int kShortColumns = 8;
template <int kThreads>
struct ShortShared {
  using Choose = ChooseShared<kThreads, kShortPages, 256>;
  double score[kShortPages];
  float rounded[kShortPages];
  float s[kShortColumns][kShortPages];  // scores of the coarse branch, then its probabilities over n_p
  float q[kShortColumns][kDim];         // scaled
  float sum[kShortColumns];
  int page[kShortPages];
  union {
    float part[kThreads / 32][kShortColumns][kDim];
    Choose choose;
  };
};

// Short requests, one CTA per (request, key/value head): score, choose, and attend over the page means.
// Half a warp scores a page; for the values a warp takes every eighth page and a lane four dims.
template <int kType, bool kCoarse, int kThreads>
__global__ void __launch_bounds__(kThreads, 512 / kThreads) page_short_kernel(const __grid_constant__ SelectParams a) {
  constexpr int kWarps = kThreads / 32;
  __shared__ __align__(16) ShortShared<kThreads> sh;
  const PagedSelectParams& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = lane >> 4, part = lane & 15;
  if (!p.early) {
    pdl_wait();
    pdl_release();
  }
  const int request = blockIdx.x / p.kv_heads, head = blockIdx.x % p.kv_heads;
  const int length = tokens_of(p, request), n = (length + kBlock - 1) / kBlock;
  const bool scoring = p.chosen != nullptr && n > p.keep;
  for (int i = tid; i < n; i += kThreads) {
    int page = p.tables[request * p.table_stride + i];
    if (page < 0 || page >= p.pages) {
      paged_error(p.status, kPagedBadPage);
      page = -1;
    }
    sh.page[i] = page;
  }
  // Dims 4 part .. 4 part + 3 and 64 more.
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + request * p.q_row_stride + static_cast<long long>(head) * p.group * p.q_head_stride;
  const auto load_q = [&](int g, float (&x)[8]) {
    const uint2* src = reinterpret_cast<const uint2*>(q + static_cast<long long>(g) * p.q_head_stride) + part;
    const uint2 lo = src[0], hi = src[16];
    const uint32_t w[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = unpack1<kType>(static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1))));
  };
  double sum_q[8] = {};
  if (scoring) {
#pragma unroll 4
    for (int g = 0; g < p.group; ++g) {
      float x[8];
      load_q(g, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum_q[i] += x[i];
    }
  }
  const auto stage_q = [&](int first_q, int columns) {
    for (int x = tid; x < columns * kDim; x += kThreads)
      sh.q[x / kDim][x % kDim] = unpack1<kType>(q[static_cast<long long>(first_q + x / kDim) * p.q_head_stride + x % kDim]) * (p.scale * kLog2e);
  };
  if (kCoarse) stage_q(0, min(kShortColumns, p.group));
  __syncthreads();
  if (p.early) {
    pdl_wait();
    pdl_release();
  }
  constexpr int kStep = 2 * kWarps;  // pages 2 warp + half + kStep * j
  for (int first_q = 0; first_q < (kCoarse ? p.group : 1); first_q += kShortColumns) {
    const int columns = min(kShortColumns, p.group - first_q);
    if (first_q > 0) {
      stage_q(first_q, columns);
      __syncthreads();
    }
    if (kCoarse || scoring) {
      for (int j0 = 0; j0 < n; j0 += 4 * kStep) {
        float k[4][8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = j0 + kStep * j + 2 * warp + half, id = i < n ? sh.page[i] : -1;
          const float4* row = reinterpret_cast<const float4*>(p.k_sum + (static_cast<long long>(max(id, 0)) * p.kv_heads + head) * kDim) + part;
          const float4 lo = id >= 0 ? row[0] : make_float4(0.f, 0.f, 0.f, 0.f), hi = id >= 0 ? row[16] : make_float4(0.f, 0.f, 0.f, 0.f);
          k[j][0] = lo.x, k[j][1] = lo.y, k[j][2] = lo.z, k[j][3] = lo.w, k[j][4] = hi.x, k[j][5] = hi.y, k[j][6] = hi.z, k[j][7] = hi.w;
        }
        if (scoring && first_q == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = j0 + kStep * j + 2 * warp + half, tokens = min(kBlock, length - i * kBlock);
            double sum = 0.;
#pragma unroll
            for (int d = 0; d < 8; ++d) sum = fma(sum_q[d], static_cast<double>(k[j][d]), sum);
#pragma unroll
            for (int d = 8; d > 0; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
            if (part == 0 && i < n) sh.score[i] = finite_score(tokens == kBlock ? sum * (1. / kBlock) : sum / static_cast<double>(tokens));
          }
        }
        if (kCoarse) {
          // The four pages' sums over 16 lanes end in lanes 0, 4, 8 and 12: pages are handed over on the way.
          const int own = 2 * ((part >> 3) & 1) + ((part >> 2) & 1), i = j0 + kStep * own + 2 * warp + half;
          const float inv = 1.f / static_cast<float>(max(min(kBlock, length - i * kBlock), 1));
          const bool live = i < n && sh.page[i < n ? i : 0] >= 0;
#pragma unroll 2
          for (int g = 0; g < columns; ++g) {
            const float4 lo = *reinterpret_cast<const float4*>(&sh.q[g][4 * part]), hi = *reinterpret_cast<const float4*>(&sh.q[g][64 + 4 * part]);
            const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            float s[4] = {};
#pragma unroll
            for (int d = 0; d < 8; ++d)
#pragma unroll
              for (int j = 0; j < 4; ++j) s[j] = fmaf(x[d], k[j][d], s[j]);
            const bool up8 = part & 8, up4 = part & 4;
            const float a0 = (up8 ? s[2] : s[0]) + __shfl_xor_sync(~0u, up8 ? s[0] : s[2], 8);
            const float a1 = (up8 ? s[3] : s[1]) + __shfl_xor_sync(~0u, up8 ? s[1] : s[3], 8);
            float sum = (up4 ? a1 : a0) + __shfl_xor_sync(~0u, up4 ? a0 : a1, 4);
            sum += __shfl_xor_sync(~0u, sum, 2);
            sum += __shfl_xor_sync(~0u, sum, 1);
            if ((part & 3) == 0 && i < n) sh.s[g][i] = live ? sum * inv : -INFINITY;
          }
        }
      }
    }
    if (!kCoarse) break;
    __syncthreads();
    for (int g = warp; g < columns; g += kWarps) {  // a warp per query head
      float top = -INFINITY, sum = 0.f;
      for (int i = lane; i < n; i += 32) top = fmaxf(top, sh.s[g][i]);
#pragma unroll
      for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      for (int i = lane; i < n; i += 32) {
        const float w = sh.page[i] < 0 ? 0.f : exp2_fast(sh.s[g][i] - finite_or_zero(top));
        sum += w;
        sh.s[g][i] = w / static_cast<float>(min(kBlock, length - i * kBlock));
      }
#pragma unroll
      for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
      if (lane == 0) sh.sum[g] = sum;
    }
    __syncthreads();
    float o[kShortColumns][4] = {};
    for (int i0 = warp; i0 < n; i0 += 4 * kWarps) {
      float4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * kWarps, id = i < n ? sh.page[i] : -1;
        v[j] = id >= 0 ? reinterpret_cast<const float4*>(p.v_sum + (static_cast<long long>(id) * p.kv_heads + head) * kDim)[lane]
                       : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * kWarps;
        if (i >= n) break;
#pragma unroll
        for (int g = 0; g < kShortColumns; ++g) {
          if (g >= columns) break;
          const float w = sh.s[g][i];
          o[g][0] = fmaf(w, v[j].x, o[g][0]), o[g][1] = fmaf(w, v[j].y, o[g][1]), o[g][2] = fmaf(w, v[j].z, o[g][2]), o[g][3] = fmaf(w, v[j].w, o[g][3]);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < kShortColumns; ++g)
      if (g < columns) *reinterpret_cast<float4*>(&sh.part[warp][g][4 * lane]) = make_float4(o[g][0], o[g][1], o[g][2], o[g][3]);
    __syncthreads();
    for (int x = tid; x < columns * kDim; x += kThreads) {
      const int g = x / kDim, d = x % kDim;
      float y = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) y += sh.part[w][g][d];
      const float sum = sh.sum[g];
      p.coarse[((static_cast<long long>(request) * p.kv_heads + head) * p.group + first_q + g) * kDim + d] = sum == 0.f ? 0.f : y / sum;
    }
    __syncthreads();
  }
  __syncthreads();
  if (p.chosen != nullptr) choose_pages(p, sh.score, sh.rounded, n, p.chosen + static_cast<long long>(blockIdx.x) * p.keep, sh.choose);
}

template <bool kCoarse, int kThreads>
cudaError_t launch_short_threads(const SelectParams& a, int tiles, cudaStream_t stream) {
  return a.p.dtype == kBf16 ? launch_overlapped<page_short_kernel<kBf16, kCoarse, kThreads>>(dim3(tiles), kThreads, 0, stream, a)
                            : launch_overlapped<page_short_kernel<kFp16, kCoarse, kThreads>>(dim3(tiles), kThreads, 0, stream, a);
}
template <bool kCoarse>
cudaError_t launch_short(const SelectParams& a, cudaStream_t stream) {
  const int tiles = a.p.requests * a.p.kv_heads;
  if (tiles > 592) return launch_short_threads<kCoarse, 64>(a, tiles, stream);
  if (tiles > 296) return launch_short_threads<kCoarse, 128>(a, tiles, stream);
  return launch_short_threads<kCoarse, 256>(a, tiles, stream);
}

// CTAs below `tiles` choose pages, one for each (request, key/value head); the others join partial
// results, `join_columns` query heads of one (request, virtual head) each.
__global__ void __launch_bounds__(kChooseThreads, 4) page_choose_kernel(const __grid_constant__ SelectParams a, int tiles, int join_columns) {
  extern __shared__ __align__(16) float rounded[];  // [width]
  __shared__ __align__(16) ChooseShared<kChooseThreads, kMostSelectPages, 2048> sh;
  const PagedSelectParams& p = a.p;
  pdl_wait();
  pdl_release();
  if (static_cast<int>(blockIdx.x) < tiles) {
    const int n = pages_of(p, blockIdx.x / p.kv_heads);
    choose_pages(p, a.score + static_cast<long long>(blockIdx.x) * p.width, rounded, n, p.chosen + static_cast<long long>(blockIdx.x) * p.keep, sh);
    return;
  }
  // Where the tile's units lie: the same split as the workers'.
  const int heads = p.kv_heads * a.chunks, parts = (a.chunk_heads + join_columns - 1) / join_columns;
  const int x = (blockIdx.x - tiles) / parts, column = (blockIdx.x - tiles) % parts * join_columns, s = x / heads, hv = x % heads;
  int before = 0, total = 0;
  for (int e = threadIdx.x; e < p.requests; e += kChooseThreads) {
    const int n = pages_of(p, e);
    total += n;
    before += e < s ? n : 0;
  }
  before = __reduce_add_sync(~0u, before), total = __reduce_add_sync(~0u, total);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sh.low[warp] = before, sh.high[warp] = total;
  __syncthreads();
  before = __reduce_add_sync(~0u, lane < kChooseWarps ? sh.low[lane] : 0), total = __reduce_add_sync(~0u, lane < kChooseWarps ? sh.high[lane] : 0);
  const int n = pages_of(p, s);
  if (n == 0) return;
  const WorkSplit split(total * heads, a.workers, kLeastUnits);
  const int begin = before * heads + hv * n, first = split.owner(begin), last = split.owner(begin + n - 1);
  if (first == last) return;
  float4(*part)[32] = reinterpret_cast<float4(*)[32]>(sh.hist);
  static_assert(sizeof(sh.hist) >= kChooseWarps * 32 * sizeof(float4), "partial sums of the warps");
  const int head = hv / a.chunks, first_q = (hv % a.chunks) * a.chunk_heads;
  const int columns_end = min(min(column + join_columns, a.chunk_heads), p.group - first_q);
  if (column >= columns_end) return;
  join_partials<kChooseWarps>(warp, 1, first, last, column, columns_end, a.chunk_heads, a.stats, a.partials, part,
                              [&](int col, float, float sum, float4 y) {
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    if (sum == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
    const long long row = (static_cast<long long>(s) * p.kv_heads + head) * p.group + first_q + col;
    *reinterpret_cast<float4*>(p.coarse + row * kDim + 4 * lane) = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
  });
}

struct Workspace {
  int64_t score, partials, stats, bytes;
};
bool is_short(int64_t tiles, int64_t width, bool coarse) { return width <= (coarse && tiles > 592 ? kShortPages / 2 : kShortPages); }
Workspace workspace_of(int64_t requests, int64_t kv_heads, int group, int64_t width, bool choose, bool coarse) {
  const int columns = group < kColumnsMax ? group : kColumnsMax;
  Workspace w{};
  if (is_short(requests * kv_heads, width, coarse)) return w;
  int64_t at = choose ? requests * kv_heads * width * 8 : 0;
  at = (at + 15) / 16 * 16;
  if (coarse) {
    w.partials = at, at += 2LL * kWorkersMax * columns * kDim * 4;
    w.stats = at, at += 2LL * kWorkersMax * columns * 8;
  }
  w.bytes = at;
  return w;
}

template <int kType, int kHeads>
cudaError_t launch(SelectParams& a, int sms, cudaStream_t stream) {
  using Shared = ScoreShared<(kHeads > 0 ? kHeads : 1), (kHeads > 0)>;
  const int ctas = sms < kWorkersMax / Shared::kWarps ? sms : kWorkersMax / Shared::kWarps;
  static_assert(Shared::kWarps * sizeof(Shared) <= 226 * 1024, "shared memory of one CTA");
  a.workers = ctas * Shared::kWarps;
  return launch_overlapped<page_scores_kernel<kType, kHeads>>(dim3(ctas), 32 * Shared::kWarps, Shared::kWarps * static_cast<int>(sizeof(Shared)), stream, a);
}
template <int kType>
cudaError_t launch_type(SelectParams& a, int sms, cudaStream_t stream) {
  if (a.p.coarse == nullptr) return launch<kType, 0>(a, sms, stream);
  if (a.chunk_heads == 1) return launch<kType, 1>(a, sms, stream);
  if (a.chunk_heads == 2) return launch<kType, 2>(a, sms, stream);
  if (a.chunk_heads == 3) return launch<kType, 3>(a, sms, stream);
  if (a.chunk_heads == 4) return launch<kType, 4>(a, sms, stream);
  if (a.chunk_heads == 5) return launch<kType, 5>(a, sms, stream);
  if (a.chunk_heads == 6) return launch<kType, 6>(a, sms, stream);
  return launch<kType, 8>(a, sms, stream);
}

}  // namespace

int64_t paged_select_workspace_bytes(int requests, int kv_heads, int group, int width, bool choose, bool coarse) {
  return workspace_of(requests, kv_heads, group, width, choose, coarse).bytes;
}

cudaError_t launch_paged_select(const PagedSelectParams& p, cudaStream_t stream) {
  SelectParams a{};
  a.p = p;
  const bool choose = p.chosen != nullptr, coarse = p.coarse != nullptr;
  if (is_short(static_cast<int64_t>(p.requests) * p.kv_heads, p.width, coarse)) return coarse ? launch_short<true>(a, stream) : launch_short<false>(a, stream);
  // Without the coarse branch one pass serves the whole group.
  a.chunks = coarse ? (p.group + kColumnsMax - 1) / kColumnsMax : 1;
  a.chunk_heads = (p.group + a.chunks - 1) / a.chunks;
  int device = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (err != cudaSuccess) return err;
  const Workspace w = workspace_of(p.requests, p.kv_heads, p.group, p.width, choose, coarse);
  a.score = reinterpret_cast<double*>(p.workspace);
  a.partials = reinterpret_cast<float*>(p.workspace + w.partials);
  a.stats = reinterpret_cast<float2*>(p.workspace + w.stats);
  err = p.dtype == kBf16 ? launch_type<kBf16>(a, sms, stream) : launch_type<kFp16>(a, sms, stream);
  if (err != cudaSuccess) return err;
  const int tiles = choose ? p.requests * p.kv_heads : 0;
  // With few tiles each of them has many partial results: a CTA then joins one query head's.
  const int all = coarse ? p.requests * p.kv_heads * a.chunks : 0;
  const int join_columns = static_cast<int64_t>(all) * a.chunk_heads <= 592 ? 1 : a.chunk_heads;
  const int joins = all * ((a.chunk_heads + join_columns - 1) / join_columns);
  return launch_overlapped<page_choose_kernel>(dim3(tiles + joins), kChooseThreads, choose ? p.width * 4 : 0, stream, a, tiles, join_columns);
}

}  // namespace vsa
