// What the kernels of paged attention share: query fragments, a warp's step over 16 keys, the output.
#pragma once
#include "vsa_paged_common.cuh"

namespace vsa {

VSA_DEVICE int tokens_of(const PagedAttentionParams& p, int s) { return min(max(p.lengths[s], 0), p.width * kBlock); }
// Units (pages) of every key/value head of request s.
VSA_DEVICE int units_of(const PagedAttentionParams& p, int s) {
  const int n = (tokens_of(p, s) + kBlock - 1) / kBlock;
  return p.chosen == nullptr ? n : min(n, p.keep);
}

template <bool kHalf>
VSA_DEVICE void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kHalf)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two FP32 values cut to 16 bits, `lo` in the low half.
template <bool kHalf>
VSA_DEVICE uint32_t truncate2(float lo, float hi) {
  uint32_t r;
  if (kHalf) asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Transposes an 8 x 8 matrix of 16-bit values held two per lane.
VSA_DEVICE uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
VSA_DEVICE uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// One warp: Q^T fragments of the eight query columns from `column0` on - column c is query head first_head + c -
// zero from `columns` on.  Lane (r, j) holds column column0 + r, its 16-byte chunks in the order in which the K
// operand takes them.
template <int kType, bool kE4m3>
VSA_DEVICE void load_queries(const PagedAttentionParams& p, uint4 (*fragments)[32], float* factors, int request, int first_head, int column0, int columns, int head) {
  const int lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3, col = column0 + r;
  const uint16_t* src = static_cast<const uint16_t*>(p.q) + request * p.q_row_stride +
                        static_cast<long long>(first_head + min(col, columns - 1)) * p.q_head_stride;
  uint32_t q[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // 16 bits: half i/2, chunk 2j + i%2, 8 dims.  8 bits: chunk 2j + i/2 of 16 dims, its half i%2.
    const int dim = kE4m3 ? 16 * (2 * j + i / 2) + 8 * (i % 2) : 64 * (i / 2) + 8 * (2 * j + i % 2);
    uint4 v = *reinterpret_cast<const uint4*>(src + dim);
    if (col >= columns) v = make_uint4(0, 0, 0, 0);
    q[4 * i] = v.x, q[4 * i + 1] = v.y, q[4 * i + 2] = v.z, q[4 * i + 3] = v.w;
  }
  float to_log2 = p.scale * kLog2e;
  if (kE4m3) {
    to_log2 *= p.k_scale[head];
    if (kType == kBf16) {
      // FP16 holds the row after its largest value is brought to [2^14, 2^15).
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 f = unpack_bf16(q[i]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      const int e = static_cast<int>(__float_as_uint(top) >> 23);  // biased exponent, 255 = infinity
      const int shift = e == 0 || e == 255 ? 0 : min(max(127 + 14 - e, -113), 100);
      const float up = __uint_as_float((127 + shift) << 23);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 f = unpack_bf16(q[i]);
        q[i] = pack2<kFp16>(f.x * up, f.y * up);
      }
      to_log2 *= __uint_as_float((127 - shift) << 23);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) fragments[i][lane] = make_uint4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
  if (j == 0) factors[r] = to_log2;
}

// Writes two neighbouring dims of an output row (normalised, with the gated merge).
template <int kType>
VSA_DEVICE void store_pair(const PagedAttentionParams& p, int request, int qh, int d, float y0, float y1) {
  const long long row = static_cast<long long>(request) * p.kv_heads * p.group + qh;
  if (p.gate != nullptr) {
    const uint32_t g = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.gate) + request * p.gate_row_stride + qh * p.gate_head_stride + d);
    const float2 c = *reinterpret_cast<const float2*>(p.coarse + row * kDim + d);
    y0 += unpack1<kType>(g & 0xFFFF) * c.x, y1 += unpack1<kType>(g >> 16) * c.y;
  }
  *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + row * kDim + d) = pack2<kType>(y0, y1);
}

// With BF16 the weighted sums of values are kept smaller by this: 2^24 keys of any BF16 values, each with the largest
// weight of 2^8, do not overflow FP32 before they are divided by the sum of the weights.
template <int kType, bool kE4m3>
constexpr float kSmaller = !kE4m3 && kType == kBf16 ? 2.3283064365386963e-10f : 1.f;  // 2^-32

// What a warp holds of eight query columns while it passes over keys; lane (r, j) columns 2j and 2j + 1.
struct Running {
  float o[8][4];  // O^T * kSmaller: [product][column and, + 2, the other row]
  float m[2];     // maximum less kShift
  float l[2];     // sum over this lane's keys
  float base[2];  // m, or 0 as long as it is -infinity
  float limit[2];  // a score (less base) above it raises the maximum

  VSA_DEVICE void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    m[0] = m[1] = limit[0] = limit[1] = -INFINITY;
    l[0] = l[1] = base[0] = base[1] = 0.f;
  }
};

// The four keys whose values lane (r, j) feeds to the second product.
VSA_DEVICE int value_key(int i, int j) { return 2 * j + (i & 1) + 8 * (i >> 1); }

// One warp takes 16 keys, the first `valid` of them seen.  `q_at(i)` are the query fragments; `k_at(upper, i)`
// chunk i of this lane's key r + 8 upper: of 16 bits chunk 2j + i % 2 of half i / 2, of 8 bits chunk 2j + i;
// `v_at(i, half)` 16-byte chunk r of the half (of 8 bits: of the row) of value row value_key(i, j).  `keys_read` is called when the
// keys are not needed any more, `values_wanted` before the first value is.
template <int kType, bool kE4m3, class Q, class K, class Read, class Wanted, class V>
VSA_DEVICE void attend_keys(Running& s, float2 to_log2, int valid, const Q& q_at, const K& k_at, const Read& keys_read,
                            const Wanted& values_wanted, const V& v_at) {
  constexpr bool kHalf = kE4m3 || kType == kFp16;
  constexpr int kPType = kHalf ? kFp16 : kBf16;
  // Probabilities come out scaled by 2^kShift; the maximum is raised when a score exceeds it by kRaise.
  constexpr float kShift = kHalf ? 11.f : 0.f, kRaise = kHalf ? 15.f : 8.f;
  constexpr float kLeast = kHalf ? 5.9604644775390625e-8f : 1.17549435e-38f;  // smallest FP16; smallest normal BF16
  constexpr float kWeight = kHalf ? kLeast : 7.8886090522101181e-31f;  // FP16: its first term is not zero; BF16: 2^-100
  const int lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
  float acc[2][4] = {};
  if (kE4m3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 q[2] = {q_at(2 * i), q_at(2 * i + 1)}, x = k_at(0, i), y = k_at(1, i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t a0 = e4m3x2_to_half2(word(x, e) & 0xFFFF), a2 = e4m3x2_to_half2(word(x, e) >> 16);
        const uint32_t a1 = e4m3x2_to_half2(word(y, e) & 0xFFFF), a3 = e4m3x2_to_half2(word(y, e) >> 16);
        mma16816<true>(acc[e & 1], a0, a1, a2, a3, word(q[e / 2], 2 * (e % 2)), word(q[e / 2], 2 * (e % 2) + 1));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 q = q_at(i), x = k_at(0, i), y = k_at(1, i);
      mma16816<kHalf>(acc[0], x.x, y.x, x.y, y.y, q.x, q.y);
      mma16816<kHalf>(acc[1], x.z, y.z, x.w, y.w, q.z, q.w);
    }
  }
  keys_read();
  // Scores in base 2, less `base`: rows are keys r and r + 8, columns query heads 2j and 2j + 1.
  float sc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc[0][i] += acc[1][i];
    sc[i] = fmaf(acc[0][i], (i & 1) ? to_log2.y : to_log2.x, -s.base[i & 1]);
  }
  if (valid < 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r + 8 * (i / 2) >= valid) sc[i] = -INFINITY;
  }
  if (__any_sync(~0u, fmaxf(sc[0], sc[2]) > s.limit[0] || fmaxf(sc[1], sc[3]) > s.limit[1])) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float top = fmaxf(sc[c], sc[c + 2]);
#pragma unroll
      for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      top = fmaxf(s.m[c], top + s.base[c] - kShift);
      const float now = finite_or_zero(top), shrink = exp2_fast(s.m[c] - now);
#pragma unroll
      for (int i = c; i < 4; i += 2)
        if (sc[i] != -INFINITY) sc[i] = fmaf(acc[0][i], (i & 1) ? to_log2.y : to_log2.x, -now);
      s.m[c] = top, s.base[c] = now;
      if (top != -INFINITY) s.limit[c] = kRaise;
      s.l[c] *= shrink;
#pragma unroll
      for (int i = 0; i < 8; ++i) s.o[i][c] *= shrink, s.o[i][c + 2] *= shrink;
    }
  }
  uint32_t hi[2], lo[2], rest[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    float p0 = exp2_fast(sc[2 * x]), p1 = exp2_fast(sc[2 * x + 1]);
    s.l[0] += p0;
    s.l[1] += p1;
    if (kE4m3) {  // e4m3 has no infinities: both terms are rounded, the second has either sign
      const uint32_t both = pack2<kFp16>(p0, p1);
      hi[x] = transpose8x8(both);
      lo[x] = transpose8x8(pack2<kFp16>(p0 - unpack1<kFp16>(both & 0xFFFF), p1 - unpack1<kFp16>(both >> 16)));
    } else {
      p0 *= kSmaller<kType, kE4m3>, p1 *= kSmaller<kType, kE4m3>;
      // No term of a key that has weight is zero; those of others may be, so that their values add what they should:
      // next to nothing.
      const float least0 = p0 >= kWeight ? kLeast : 0.f, least1 = p1 >= kWeight ? kLeast : 0.f;
      const uint32_t both = truncate2<kHalf>(p0, p1);
      const float r0 = fmaxf(p0 - unpack1<kPType>(both & 0xFFFF), least0), r1 = fmaxf(p1 - unpack1<kPType>(both >> 16), least1);
      hi[x] = transpose8x8(both);
      if (kHalf) {
        lo[x] = transpose8x8(pack2<kPType>(r0, r1));
      } else {
        const uint32_t next = truncate2<kHalf>(r0, r1);
        lo[x] = transpose8x8(next);
        rest[x] = transpose8x8(pack2<kPType>(fmaxf(r0 - unpack1<kPType>(next & 0xFFFF), least0), fmaxf(r1 - unpack1<kPType>(next >> 16), least1)));
      }
    }
  }
  values_wanted();
  // V^T: rows are dims, columns keys; this lane's keys are 2j, 2j+1, 2j+8, 2j+9.
  const auto clear_rows = [&](uint4 (&v)[4]) {  // what is behind the request's last token
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (value_key(i, j) >= valid) v[i] = make_uint4(0, 0, 0, 0);
  };
  if (kE4m3) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = v_at(i, 0);
    }
    if (valid < 16) clear_rows(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // rows r: dim 16 r + 2 i, rows r + 8: dim 16 r + 2 i + 1
      const uint32_t pick = (i & 1) ? 0x7362u : 0x5140u;
      const uint32_t x = __byte_perm(word(v[0], i / 2), word(v[1], i / 2), pick);
      const uint32_t y = __byte_perm(word(v[2], i / 2), word(v[3], i / 2), pick);
      const uint32_t a0 = e4m3x2_to_half2(x & 0xFFFF), a1 = e4m3x2_to_half2(x >> 16);
      const uint32_t a2 = e4m3x2_to_half2(y & 0xFFFF), a3 = e4m3x2_to_half2(y >> 16);
      mma16816<true>(s.o[i], a0, a1, a2, a3, hi[0], hi[1]);
      mma16816<true>(s.o[i], a0, a1, a2, a3, lo[0], lo[1]);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = v_at(i, h);
      }
      if (valid < 16) clear_rows(v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // rows r: dim 64 h + 8 r + 2 e, rows r + 8: the next dim
        const uint32_t a0 = __byte_perm(word(v[0], e), word(v[1], e), 0x5410u), a1 = __byte_perm(word(v[0], e), word(v[1], e), 0x7632u);
        const uint32_t a2 = __byte_perm(word(v[2], e), word(v[3], e), 0x5410u), a3 = __byte_perm(word(v[2], e), word(v[3], e), 0x7632u);
        mma16816<kHalf>(s.o[4 * h + e], a0, a1, a2, a3, hi[0], hi[1]);
        mma16816<kHalf>(s.o[4 * h + e], a0, a1, a2, a3, lo[0], lo[1]);
        if (!kHalf) mma16816<kHalf>(s.o[4 * h + e], a0, a1, a2, a3, rest[0], rest[1]);
      }
    }
  }
}

// A lane's two neighbouring dims of product i, rows r and r + 8.
template <bool kE4m3>
VSA_DEVICE int dim_of(int i, int r) { return kE4m3 ? 16 * r + 2 * i : 64 * (i / 4) + 8 * r + 2 * (i % 4); }

}  // namespace vsa
