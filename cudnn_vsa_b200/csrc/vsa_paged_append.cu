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
// e4m3 cache, 922 MB: 161 us (5.7 TB/s), bound by the conversions as much.  One token for each of 64
// requests: 3.4 us.
#include "vsa_paged_common.cuh"

namespace vsa {

namespace {

constexpr int kThreads = 128;

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

struct Scale {
  float scale, up, down;  // the inverse, 2^-21 of it more and less
  bool divide;            // the inverse is not exact enough
};

template <int kType, bool kE4m3>
struct RowChunk {  // eight dims of one row
  uint4 raw;

  VSA_DEVICE void load_new(const char* at) { raw = load128(at); }
  VSA_DEVICE void load_old(const char* at) {
    if (kE4m3) {
      const uint2 v = load64(at);
      raw = make_uint4(v.x, v.y, 0, 0);
    } else {
      raw = load128(at);
    }
  }
  // New values as the cache holds them.
  VSA_DEVICE void store(char* at, const Scale& scale) {
    if (kE4m3) {
      // x / scale, rounded to FP32, lies between x * up and x * down: the inverse, its factor, the product and
      // the quotient itself are each off by at most 2^-24, together by at most half of 2^-21.  Where both are the
      // same number in e4m3, that is its rounding; else - one value in 65,536 - the row's chunk is divided.  Zeros,
      // infinities and NaN come out of both products.
      float x[8];
      unpack8<kType>(raw, x);
      uint32_t w[2], other = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[i] = rounded4(x + 4 * i, scale.down);
        other |= w[i] ^ rounded4(x + 4 * i, scale.up);
      }
      if (other != 0 || scale.divide) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = __fdiv_rn(x[4 * i + e], scale.scale);
          w[i] = rounded4(q, 1.f);
        }
      }
      raw = make_uint4(w[0], w[1], 0, 0);
      *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
    } else {
      *reinterpret_cast<uint4*>(at) = raw;
    }
  }
  static VSA_DEVICE uint32_t rounded4(const float* x, float factor) {
    const uint32_t lo = floats_to_e4m3x2(x[0] * factor, x[1] * factor), hi = floats_to_e4m3x2(x[2] * factor, x[3] * factor);
    return lo | (hi << 16);
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
__global__ void __launch_bounds__(kThreads, 8) paged_append_kernel(PagedAppendParams p) {
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
  Scale scale{1.f, 1.f, 1.f, false};
  if (kE4m3) {
    scale.scale = (values ? p.v_scale : p.k_scale)[head];
    const float inverse = 1.f / scale.scale;
    scale.up = inverse * (1.f + 4.76837158203125e-7f), scale.down = inverse * (1.f - 4.76837158203125e-7f);
    scale.divide = !(scale.scale > 1e-37f && scale.scale < 1e37f);
  }
  // Where this thread's first row is, or would be.
  const char* from = static_cast<const char*>(rows) + 2 * ((run.x + static_cast<long long>(group - run.w)) * row_stride + head * head_stride + 8 * chunk);
  constexpr int kRowBytes = kDim * (kE4m3 ? 1 : 2);
  char* at = static_cast<char*>(cache) + (tile + group) * kRowBytes + chunk * (kRowBytes / 16);
  RowChunk<kType, kE4m3> x[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = group + kGroups * i;
    if (row >= filled) continue;
    if (row >= run.w) x[i].load_new(from + i * (2 * kGroups * row_stride));
    else x[i].load_old(at + i * (kGroups * kRowBytes));
  }
  float acc[8] = {};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = group + kGroups * i;
    if (row >= filled) continue;
    if (row >= run.w) x[i].store(at + i * (kGroups * kRowBytes), scale);
    x[i].add_to(acc, scale.scale);
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

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams& p, cudaStream_t stream) {
  const dim3 grid(p.max_runs, p.kv_heads, 2);  // keys, values
  const bool e4m3 = p.cache_dtype == kE4m3;
  if (p.dtype == kBf16) {
    if (e4m3) return launch_overlapped<paged_append_kernel<kBf16, true>>(grid, kThreads, 0, stream, p);
    return launch_overlapped<paged_append_kernel<kBf16, false>>(grid, kThreads, 0, stream, p);
  }
  if (e4m3) return launch_overlapped<paged_append_kernel<kFp16, true>>(grid, kThreads, 0, stream, p);
  return launch_overlapped<paged_append_kernel<kFp16, false>>(grid, kThreads, 0, stream, p);
}

}  // namespace vsa
