// New key/value rows into their pages, and the sums of the pages they touch.
//
//   cache[page, h, row] = stored(x)          16 bits: x itself; e4m3: round(x / scale[h])
//   sum[page, h, :]     = sum of the page's filled rows as the cache holds them, in FP32
//
// The sum of a touched page is formed anew from ALL its rows, not added to the old sum: at most 63
// old rows (16 KiB per head) are read again, and in return the call can be repeated, a request can
// be cut back to a shorter length before the next append, and no rounding piles up over 64 steps.
// The order of the sum is fixed (the rows of a thread, then the row groups), so results do not
// depend on timing.
//
// Bound by HBM: a prompt's rows are read and written once.  One CTA takes one run (the rows that
// one request puts into one page) of one head's keys or values, 16 lanes to a row; a thread's eight
// 16-byte loads are all in flight before the first is used, 128 KiB on an SM.  113,648 rows of 12
// heads, 1.42 GB: 221 us (6.4 TB/s; 246 us with keys and values in one CTA).  100,000 such rows into an
// e4m3 cache, 922 MB: 185 us (5.0 TB/s); the conversions' chains do not hide behind so few bytes.  One
// token for each of 64 requests: 3.3 us.
#include "vsa_paged_common.cuh"

namespace vsa {

namespace {


// Loads that the compiler may not issue again instead of keeping their results: in the e4m3 kernel it did, and
// every row came from L1 or L2 once more (276 us against 199 for 100,000 rows of 12 heads).
VSA_DEVICE uint4 load128(const void* x) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(x) : "memory");
  return v;
}
VSA_DEVICE uint2 load64(const void* x) {
  uint2 v;
  asm volatile("ld.global.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(x) : "memory");
  return v;
}

template <int kType, bool kE4m3>
struct RowChunk {  // eight dims of one row
  uint4 raw;

  VSA_DEVICE void load_new(const void* x, long long at) {
    raw = load128(static_cast<const uint16_t*>(x) + at);
  }
  VSA_DEVICE void load_old(const void* cache, long long at) {
    if (kE4m3) {
      const uint2 v = load64(static_cast<const uint8_t*>(cache) + at);
      raw = make_uint4(v.x, v.y, 0, 0);
    } else {
      raw = load128(static_cast<const uint16_t*>(cache) + at);
    }
  }
  // New values as the cache holds them.
  VSA_DEVICE void store(void* cache, long long at, float scale, float inverse) {
    if (kE4m3) {
      float x[8];
      unpack8<kType>(raw, x);
      uint32_t w[2];
      // x / scale rounds like x * inverse (off by two units in the last place at most) unless a
      // border between two e4m3 values lies that near.  Borders and values have four significant
      // bits, so their low 19 fraction bits are zero; every number within four units of such a one - 1 in
      // 65,536, and exact quotients - is divided.
      float q[8];
      unsigned least = ~0u;  // of the low 19 bits, after four are added, in the upper bits
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[i] = x[i] * inverse;
        least = min(least, __float_as_uint(q[i]) * 8192u + 4u * 8192u);
      }
      if (least < 8u * 8192u || !(scale > 1e-37f && scale < 1e37f)) {  // or the inverse is not exact enough
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(x[i], scale);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t lo = floats_to_e4m3x2(q[4 * i], q[4 * i + 1]);
        const uint32_t hi = floats_to_e4m3x2(q[4 * i + 2], q[4 * i + 3]);
        w[i] = lo | (hi << 16);
      }
      raw = make_uint4(w[0], w[1], 0, 0);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(cache) + at) = make_uint2(w[0], w[1]);
    } else {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(cache) + at) = raw;
    }
  }
  VSA_DEVICE void add_to(float (&acc)[8], float scale) const {
    if (kE4m3) {
      const uint32_t w[2] = {raw.x, raw.y};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = e4m3x2_to_floats(static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2))));
        acc[2 * i] += f.x * scale;
        acc[2 * i + 1] += f.y * scale;
      }
    } else {
      float x[8];
      unpack8<kType>(raw, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += x[i];
    }
  }
};

template <int kType, bool kE4m3, int kThreads, int kResident>
__global__ void __launch_bounds__(kThreads, kResident) paged_append_kernel(PagedAppendParams p) {
  constexpr int kGroups = kThreads / 16, kRows = kBlock / kGroups;  // rows that are worked on at a time; of a thread
  __shared__ __align__(16) float part[kThreads / 32][kDim];
  pdl_wait();
  pdl_release();
  const int4 run = p.runs[blockIdx.x];  // {first row, rows, page, first row in the page}
  if (run.y <= 0) return;
  const int filled = run.w + run.y;
  if (run.z < 0 || run.z >= p.pages || run.w < 0 || filled > kBlock || run.x < 0 || run.x + static_cast<long long>(run.y) > p.tokens) {
    if (threadIdx.x == 0) paged_error(p.status, kPagedBadPage);
    return;
  }
  const int head = blockIdx.y, chunk = threadIdx.x % 16, group = threadIdx.x / 16;
  const bool values = blockIdx.z != 0;
  const void* rows = values ? p.v : p.k;
  void* cache = values ? p.v_cache : p.k_cache;
  const long long row_stride = values ? p.v_row_stride : p.k_row_stride, head_stride = values ? p.v_head_stride : p.k_head_stride;
  const long long tile = (static_cast<long long>(run.z) * p.kv_heads + head) * kBlock;
  const float scale = kE4m3 ? (values ? p.v_scale : p.k_scale)[head] : 1.f, inverse = kE4m3 ? 1.f / scale : 1.f;
  RowChunk<kType, kE4m3> x[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = group + kGroups * i;
    if (row >= filled) continue;
    if (row >= run.w) x[i].load_new(rows, (run.x + static_cast<long long>(row - run.w)) * row_stride + head * head_stride + 8 * chunk);
    else x[i].load_old(cache, (tile + row) * kDim + 8 * chunk);
  }
  float acc[8] = {};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = group + kGroups * i;
    if (row >= filled) continue;
    if (row >= run.w) x[i].store(cache, (tile + row) * kDim + 8 * chunk, scale, inverse);
    x[i].add_to(acc, scale);
  }
  // Two row groups per warp, then the warps.
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] += __shfl_xor_sync(~0u, acc[i], 16);
  const int warp = threadIdx.x / 32;
  if ((threadIdx.x & 31) < 16) {
    *reinterpret_cast<float4*>(&part[warp][8 * chunk]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    *reinterpret_cast<float4*>(&part[warp][8 * chunk + 4]) = make_float4(acc[4], acc[5], acc[6], acc[7]);
  }
  __syncthreads();
  if (threadIdx.x >= kDim) return;
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) sum += part[w][threadIdx.x];
  (values ? p.v_sum : p.k_sum)[(static_cast<long long>(run.z) * p.kv_heads + head) * kDim + threadIdx.x] = sum;
}

template <int kType>
cudaError_t launch(const PagedAppendParams& p, dim3 grid, cudaStream_t stream) {
  if (p.cache_dtype != kE4m3) return launch_overlapped<paged_append_kernel<kType, false, 128, 8>>(grid, 128, 0, stream, p);
  // Rounding to 8 bits is a long chain: runs of many rows, too few to fill the SMs more than three times, take
  // twice the threads (16 requests of 4 heads with 1,000 rows each 14.3 : 15.3 us, of 8 heads with 100 rows 4.9 : 6.5;
  // but 118 requests of 12 heads with two rows 10.1 : 8.3, 64 of 8 heads with 1,000 rows 88.7 : 82.9).
  if (p.tokens > 4LL * p.max_runs && static_cast<long long>(p.max_runs) * p.kv_heads <= 2048)
    return launch_overlapped<paged_append_kernel<kType, true, 256, 4>>(grid, 256, 0, stream, p);
  return launch_overlapped<paged_append_kernel<kType, true, 128, 8>>(grid, 128, 0, stream, p);
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams& p, cudaStream_t stream) {
  const dim3 grid(p.max_runs, p.kv_heads, 2);  // keys, values
  return p.dtype == kBf16 ? launch<kBf16>(p, grid, stream) : launch<kFp16>(p, grid, stream);
}

}  // namespace vsa
