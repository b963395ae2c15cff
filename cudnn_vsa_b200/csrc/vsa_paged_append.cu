// New key/value rows into their pages, and the sums of the pages they touch.
//
//   cache[page, h, row] = stored(x)          16 bits: x itself; e4m3: round(x / scale[h])
//   sum[page, h, :]     = sum of the page's filled rows as the cache holds them, in FP32
//
// The sum of a touched page is formed anew from ALL its rows, not added to the old sum: at most 63
// old rows (16 KiB per head) are read again, and in return the call can be repeated, a request can
// be cut back to a shorter length before the next append, and no rounding piles up over 64 steps.
// The order of the sum is fixed (four rows per thread, then 16 row groups), so results do not
// depend on timing.
//
// Bound by HBM: a prompt's rows are read and written once.  One CTA takes one run (the rows that
// one request puts into one page) of one head's keys or values, 16 lanes to a row, 16 rows at a
// time; a thread's four 16-byte loads are all in flight before the first is used, and six CTAs to an
// SM hold 96 KiB in flight.  113,648 rows of 12 heads, 1.42 GB: 221 us (6.4 TB/s; 246 us with keys and
// values in one CTA, which left three to an SM).  One token for each of 64 requests: 3.6 us.
#include "vsa_paged_common.cuh"

namespace vsa {

namespace {

constexpr int kAppendThreads = 256;

template <int kType, bool kE4m3>
struct RowChunk {  // eight dims of one row
  uint4 raw;

  VSA_DEVICE void load_new(const void* x, long long at) {
    raw = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at);
  }
  VSA_DEVICE void load_old(const void* cache, long long at) {
    if (kE4m3) {
      const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(cache) + at);
      raw = make_uint4(v.x, v.y, 0, 0);
    } else {
      raw = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(cache) + at);
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
      bool near = !(scale > 1e-37f && scale < 1e37f);  // the inverse is not exact enough
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[i] = x[i] * inverse;
        near |= ((__float_as_uint(q[i]) + 4) & 0x7FFF8) == 0;
      }
      if (near) {
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

template <int kType, bool kE4m3>
__global__ void __launch_bounds__(kAppendThreads, kE4m3 ? 5 : 6) paged_append_kernel(PagedAppendParams p) {
  __shared__ __align__(16) float part[kAppendThreads / 32][kDim];
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
  RowChunk<kType, kE4m3> x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = group + 16 * i;
    if (row >= filled) continue;
    if (row >= run.w) x[i].load_new(rows, (run.x + static_cast<long long>(row - run.w)) * row_stride + head * head_stride + 8 * chunk);
    else x[i].load_old(cache, (tile + row) * kDim + 8 * chunk);
  }
  float acc[8] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = group + 16 * i;
    if (row >= filled) continue;
    if (row >= run.w) x[i].store(cache, (tile + row) * kDim + 8 * chunk, scale, inverse);
    x[i].add_to(acc, scale);
  }
  // Two row groups per warp, then the eight warps.
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
  for (int w = 0; w < kAppendThreads / 32; ++w) sum += part[w][threadIdx.x];
  (values ? p.v_sum : p.k_sum)[(static_cast<long long>(run.z) * p.kv_heads + head) * kDim + threadIdx.x] = sum;
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams& p, cudaStream_t stream) {
  const dim3 grid(p.max_runs, p.kv_heads, 2);  // keys, values
  const bool e4m3 = p.cache_dtype == kE4m3;
  if (p.dtype == kBf16) {
    if (e4m3) return launch_overlapped<paged_append_kernel<kBf16, true>>(grid, kAppendThreads, 0, stream, p);
    return launch_overlapped<paged_append_kernel<kBf16, false>>(grid, kAppendThreads, 0, stream, p);
  }
  if (e4m3) return launch_overlapped<paged_append_kernel<kFp16, true>>(grid, kAppendThreads, 0, stream, p);
  return launch_overlapped<paged_append_kernel<kFp16, false>>(grid, kAppendThreads, 0, stream, p);
}

}  // namespace vsa
