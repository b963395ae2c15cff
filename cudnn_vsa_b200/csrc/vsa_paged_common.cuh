// Element conversions shared by the paged-cache kernels.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

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

VSA_DEVICE void paged_error(int* status, int code) {
  if (status != nullptr) atomicCAS(status, 0, code);
}

}  // namespace vsa
