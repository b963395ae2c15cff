// Element conversions shared by the paged-cache kernels.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>
#include <mutex>

#include "vsa_common.cuh"
#include "vsa_paged.h"

namespace vsa {

// Eight 16-bit values (bf16 or fp16) <-> FP32.
template <int kType>
VSA_DEVICE void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    if (kType == kBf16) {
      f = unpack_bf16(w[i]);
    } else {
      f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <int kType>
VSA_DEVICE uint32_t pack2(float lo, float hi) {
  if (kType == kBf16) return pack_bf16(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int kType>
VSA_DEVICE float unpack1(uint16_t v) {
  if (kType == kBf16) return __uint_as_float(static_cast<uint32_t>(v) << 16);
  return __half2float(*reinterpret_cast<const __half*>(&v));
}

// Two e4m3 values as half2: exact, every e4m3 value is an fp16 value.
VSA_DEVICE uint32_t e4m3x2_to_half2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
// Two FP32 values rounded to e4m3, saturated at +-448; `lo` in the low byte.
VSA_DEVICE uint16_t floats_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
VSA_DEVICE float2 e4m3x2_to_floats(uint16_t v) {
  const uint32_t h = e4m3x2_to_half2(v);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

VSA_DEVICE float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
VSA_DEVICE float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Programmatic stream serialisation: a kernel launched this way starts while its predecessor still
// runs.  Every thread waits before it reads what the predecessor may write and before it writes;
// `pdl_release` lets the successor start, which waits in turn.  Every kernel here waits before it
// releases, so that when one starts, all work before its predecessor is complete: where the
// predecessor is known (the kernels of one decode step), it reads older inputs - q, tables, lengths -
// before it waits.  A kernel by itself may follow any other: a plan that is still writing lengths and
// tables, a kernel that is writing q.  So all inputs are read with plain loads, which stay behind the wait; loads
// marked read-only for the whole kernel (ld.global.nc) may be moved ahead of it or find a stale line.
VSA_DEVICE void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
VSA_DEVICE void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Work split.  The units (pages) of all (request, virtual head) tiles are numbered in that order, and
// worker w takes `each` consecutive ones, the first `extra` workers one more.  A range covers the end
// of one tile, whole tiles and the start of another.
struct WorkSplit {
  int total, workers, each, extra;
  WorkSplit() = default;
  // At least `least` units for each worker that has any.
  VSA_DEVICE WorkSplit(int units, int most_workers, int least) : total(units) {
    workers = max(min(most_workers, total / least), 1);
    each = total / workers;
    extra = total - each * workers;
  }
  VSA_DEVICE int begin(int worker) const { return worker * each + min(worker, extra); }
  VSA_DEVICE int owner(int unit) const {
    const int big = extra * (each + 1);
    return unit < big ? unit / (each + 1) : extra + (unit - big) / each;
  }
};
struct WorkRange {
  int begin, end;           // units
  int request, head, unit;  // where `begin` lies
};
// All lanes of a warp call this together: lane l sums up a contiguous part of the requests.
// `units(s)` are request s's units per head; workers get at least `least` units each.
template <class Units>
VSA_DEVICE WorkRange find_work(const Units& units, int requests, int heads, int worker, int workers, int least, WorkSplit& split) {
  const int lane = threadIdx.x & 31, each = (requests + 31) / 32;
  const int first = min(lane * each, requests), last = min(first + each, requests);
  int mine = 0;
  for (int s = first; s < last; ++s) mine += units(s);
  int after = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int y = __shfl_up_sync(~0u, after, d);
    if (lane >= d) after += y;
  }
  split = WorkSplit(__shfl_sync(~0u, after, 31) * heads, workers, least);
  WorkRange r{0, 0, 0, 0, 0};
  if (worker >= split.workers || split.total == 0) return r;
  r.begin = split.begin(worker);
  r.end = split.begin(worker + 1);
  const int owner = __popc(__ballot_sync(~0u, after * heads <= r.begin));  // lanes whose parts end before
  int before = __shfl_sync(~0u, after - mine, owner) * heads;
  if (each == 1) {  // the lane's part is one request
    const int count = __shfl_sync(~0u, mine, owner);
    r.request = owner;
    r.head = (r.begin - before) / count;
    r.unit = r.begin - before - r.head * count;
    return r;
  }
  for (int base = owner * each;; base += 32) {
    const int s = base + lane;
    const int n = s < requests ? units(s) : 0;
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int y = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += y;
    }
    const int found = __popc(__ballot_sync(~0u, before + upto * heads <= r.begin));
    if (found < 32 || base + 32 >= requests) {
      const int at = min(found, 31);
      const int skip = r.begin - before - __shfl_sync(~0u, upto - n, at) * heads;
      const int count = max(__shfl_sync(~0u, n, at), 1);
      r.request = base + at;
      r.head = skip / count;
      r.unit = skip - r.head * count;
      return r;
    }
    before += __shfl_sync(~0u, upto, 31) * heads;
  }
}

// Joins the workers' partial results of columns [column, columns_end) of one tile, kWarps warps that meet at
// named barrier `barrier`.  The tile starts in worker `first` (slot 2 * first + 1) and goes on through worker
// `last` (slots 2 * w); a slot has `columns_pitch` columns of 128 floats and (maximum, sum) pairs.  With
// fewer columns than warps, several warps share a column's partial results.  Latency is all that counts: the
// results, and the pairs of up to 64 workers, are fetched at once.  `store(col, top, sum, y)` gets four
// dims per lane, unnormalised.
template <int kWarps, class Store>
VSA_DEVICE void join_partials(int warp, int barrier, int first, int last, int column, int columns_end, int columns_pitch,
                              const float2* stats, const float* partials, float4 (*part)[32], const Store& store) {
  constexpr int kAhead = 6;
  const int lane = threadIdx.x & 31, columns = columns_end - column, count = last - first + 1;
  const int shares = columns < kWarps ? kWarps / columns : 1, step = kWarps / shares, share = warp % shares;
  for (int base = 0; base < columns; base += step) {
    const int col = column + base + warp / shares;
    const bool mine = warp < shares * step && col < columns_end;
    const auto slot_of = [&](int i) { return (2LL * (first + i) + (i == 0 ? 1 : 0)) * columns_pitch + col; };
    float top = -INFINITY, sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine) {
      const float2 none = make_float2(-INFINITY, 0.f);
      const float2 s0 = lane < count ? stats[slot_of(lane)] : none, s1 = lane + 32 < count ? stats[slot_of(lane + 32)] : none;
      float4 v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int x = share + i * shares;
        v[i] = x < count ? *reinterpret_cast<const float4*>(partials + slot_of(x) * kDim + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      top = fmaxf(s0.x, s1.x);
      for (int i = 64 + lane; i < count; i += 32) top = fmaxf(top, stats[slot_of(i)].x);
#pragma unroll
      for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      const float base2 = finite_or_zero(top), f0 = exp2_fast(s0.x - base2), f1 = exp2_fast(s1.x - base2);
      sum = f0 * s0.y + f1 * s1.y;
      for (int i = 64 + lane; i < count; i += 32) {
        const float2 st = stats[slot_of(i)];
        sum += exp2_fast(st.x - base2) * st.y;
      }
#pragma unroll
      for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int x = share + i * shares;
        const float lo = __shfl_sync(~0u, f0, x & 31), hi = __shfl_sync(~0u, f1, x & 31);
        float f = x < 32 ? lo : hi;
        if (x >= 64 && x < count) f = exp2_fast(stats[slot_of(x)].x - base2);
        if (x < count) y.x += f * v[i].x, y.y += f * v[i].y, y.z += f * v[i].z, y.w += f * v[i].w;
      }
#pragma unroll 4
      for (int x = share + kAhead * shares; x < count; x += shares) {
        const float4 more = *reinterpret_cast<const float4*>(partials + slot_of(x) * kDim + 4 * lane);
        const float f = exp2_fast(stats[slot_of(x)].x - base2);
        y.x += f * more.x, y.y += f * more.y, y.z += f * more.z, y.w += f * more.w;
      }
    }
    if (shares > 1) {
      part[warp][lane] = y;
      named_barrier(barrier, 32 * kWarps);
      if (mine && share == 0)
        for (int w = 1; w < shares; ++w) {
          const float4 v = part[warp + w][lane];
          y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
        }
      named_barrier(barrier, 32 * kWarps);
    }
    if (mine && share == 0) store(col, top, sum, y);
  }
}

VSA_DEVICE void paged_error(int* status, int code) {
  if (status != nullptr) atomicCAS(status, 0, code);
}

// Raises the kernel's limit of dynamic shared memory on the current device when a launch needs more than an
// earlier one asked for.  A limit never falls: another thread's launch may rely on it.
template <auto kKernel>
cudaError_t allow_shared(int smem) {
  static std::atomic<int> granted[64];
  if (smem <= 16 * 1024) return cudaSuccess;
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  if (device < 64 && granted[device].load(std::memory_order_acquire) >= smem) return cudaSuccess;
  static std::mutex raising;
  const std::lock_guard<std::mutex> lock(raising);
  if (device < 64 && granted[device].load(std::memory_order_relaxed) >= smem) return cudaSuccess;
  err = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (err == cudaSuccess && device < 64) granted[device].store(smem, std::memory_order_release);
  return err;
}

// Launch with programmatic stream serialisation.
template <auto kKernel, class Params, class... More>
cudaError_t launch_overlapped(dim3 grid, int threads, int smem, cudaStream_t stream, const Params& params, More... more) {
  const cudaError_t err = allow_shared<kKernel>(smem);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kKernel, params, more...);
}

}  // namespace vsa
