// Attention of one new token per request over its pages, or over the selected ones.
//
//   out_g = softmax(scale * q_g . K) V  [+ gate_g * coarse_g],   lse_g = log sum exp(scale * q_g . K)
//
// The simplest form: one warp per (request, query head), four dims per lane, one key at a time.
#include "vsa_paged_common.cuh"

namespace vsa {

namespace {

template <int kType, bool kE4m3>
__global__ void __launch_bounds__(32) paged_attention_kernel(PagedAttentionParams p) {
  const int request = blockIdx.y, qh = blockIdx.x, head = qh / p.group, lane = threadIdx.x;
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + request * p.q_row_stride + qh * p.q_head_stride + 4 * lane;
  float x[4], o[4] = {};
  for (int i = 0; i < 4; ++i) x[i] = unpack1<kType>(q[i]) * p.scale * (kE4m3 ? p.k_scale[head] : 1.f);
  float m = -INFINITY, l = 0.f;
  const int length = min(max(p.lengths[request], 0), p.width * kBlock);
  const int n = (length + kBlock - 1) / kBlock;
  const int32_t* chosen = p.chosen == nullptr ? nullptr : p.chosen + (static_cast<long long>(request) * p.kv_heads + head) * p.keep;
  const int count = chosen == nullptr ? n : p.keep;
  for (int c = 0; c < count; ++c) {
    const int logical = chosen == nullptr ? c : chosen[c];
    if (logical < 0 || logical >= n) continue;
    const int page = p.tables[request * p.table_stride + logical];
    if (page < 0 || page >= p.pages) {
      if (lane == 0) paged_error(p.status, kPagedBadPage);
      continue;
    }
    const long long tile = (static_cast<long long>(page) * p.kv_heads + head) * kBlock;
    for (int row = 0; row < min(kBlock, length - logical * kBlock); ++row) {
      const long long at = (tile + row) * kDim + 4 * lane;
      float k[4], v[4], s = 0.f;
      for (int i = 0; i < 4; ++i) {
        if (kE4m3) {
          k[i] = e4m3x2_to_floats(static_cast<const uint8_t*>(p.k_cache)[at + i]).x;
          v[i] = e4m3x2_to_floats(static_cast<const uint8_t*>(p.v_cache)[at + i]).x;
        } else {
          k[i] = unpack1<kType>(static_cast<const uint16_t*>(p.k_cache)[at + i]);
          v[i] = unpack1<kType>(static_cast<const uint16_t*>(p.v_cache)[at + i]);
        }
        s += x[i] * k[i];
      }
      for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(~0u, s, d);
      const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
      const float shrink = expf(m - base), w = expf(s - base);
      m = top;
      l = l * shrink + w;
      for (int i = 0; i < 4; ++i) o[i] = o[i] * shrink + w * v[i];
    }
  }
  const long long row = static_cast<long long>(request) * p.kv_heads * p.group + qh;
  for (int i = 0; i < 4; ++i) {
    const int d = 4 * lane + i;
    float y = l == 0.f ? 0.f : o[i] / l * (kE4m3 ? p.v_scale[head] : 1.f);
    if (p.gate != nullptr)
      y += unpack1<kType>(static_cast<const uint16_t*>(p.gate)[request * p.gate_row_stride + qh * p.gate_head_stride + d]) * p.coarse[row * kDim + d];
    static_cast<uint16_t*>(p.out)[row * kDim + d] = static_cast<uint16_t>(pack2<kType>(y, 0.f));
  }
  if (lane == 0 && p.lse != nullptr) p.lse[row] = m + logf(l);
}

}  // namespace

int64_t paged_workspace_bytes(int group) { return 16 * group; }

cudaError_t launch_paged_attention(const PagedAttentionParams& p, cudaStream_t stream) {
  const dim3 grid(p.kv_heads * p.group, p.requests);
  const bool e4m3 = p.cache_dtype == kE4m3;
  if (p.dtype == kBf16) {
    if (e4m3) paged_attention_kernel<kBf16, true><<<grid, 32, 0, stream>>>(p);
    else paged_attention_kernel<kBf16, false><<<grid, 32, 0, stream>>>(p);
  } else {
    if (e4m3) paged_attention_kernel<kFp16, true><<<grid, 32, 0, stream>>>(p);
    else paged_attention_kernel<kFp16, false><<<grid, 32, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace vsa
