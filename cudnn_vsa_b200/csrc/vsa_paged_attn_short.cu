// Attention of one new token per request over few pages: one CTA per (request, key/value head, eight
// query heads), nothing to join between CTAs.
//
// The mathematics and the products are those of vsa_paged_attn.cu.  There a request's pages pass through
// a ring that one CTA per SM keeps full, which costs every tile the length of its chain of steps; here
// many tiles share an SM and hide each other's chains.  A warp takes 16 keys at a time straight from
// global memory into the registers that the products read: the four lanes of a key take 32 bytes each (K),
// eight lanes the 128 bytes of a key's half (V), all eight or sixteen loads in flight at once, 8 KiB a warp,
// 16 warps to an SM.  The warps' results meet in shared memory.
//
// Time against the split kernel, us, BF16 with 4 query heads to a key/value head (e4m3 with 8), tiles of equal
// length unless said:
//       8 tiles    8 pages  7.3 :  9.6 (5.6 : 9.9)   12 pages  9.2 :  9.8 (6.6 : 10.1)   16 pages 11.4 : 9.9 (7.7 : 10.6)
//      80 tiles    8 pages  8.0 : 13.6 (6.0 : 13.4)  16 pages 14.1 : 18.0 (8.3 : 15.7)   32 pages 23.9 : 23.9 (14.0 : 19.7)
//     320 tiles    8 pages 21.7 : 24.9 (13.9 : 21.3) 16 pages 38.9 : 38.2 (23.2 : 27.8)  32 pages 72.9 : 62.2 (41.5 : 40.4)
//          ragged          18.8 : 22.1 (10.9 : 18.6)          33.0 : 26.6 (19.4 : 25.2)           47 : 39 (24.3 : 29.3)
//   1,600 tiles    8 pages 70.5 : 75.4 (42.6 : 50.0) 16 pages  130 : 134 (74.0 : 78.3)
//          ragged          42.7 : 60.6 (27.4 : 47.1)          75.5 : 81.0 (45.1 : 70.1)
#include "vsa_paged_attn.cuh"

namespace vsa {

namespace {

constexpr int kMostPages = 32;
// In the order written: the compiler spreads plain loads over the products to save registers, and then the
// keys' and values' latencies add up (512 tiles of 8 pages: 29.8 : 25.0 us).
VSA_DEVICE uint4 load128(const void* x) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(x) : "memory");
  return v;
}
int chunks_of(int group) { return (group + 7) / 8; }  // parts of up to eight query heads

template <int kWarps>
struct ShortShared {
  float2 part[kWarps][2][8][32];  // O^T fragments: column parity, product, lane
  uint4 q[4][32];
  float to_log2[8];
  float m[kWarps][8], l[kWarps][8], f[kWarps][8], top[8];
  int row[kMostPages], valid[kMostPages];  // of each page: its first cache row, its tokens (0 = left out)
};

template <int kType, bool kE4m3, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps < 16 ? 16 / kWarps : 1) paged_short_attention_kernel(PagedAttentionParams p, int chunks, int chunk_heads) {
  extern __shared__ __align__(16) uint8_t raw[];
  ShortShared<kWarps>& sh = *reinterpret_cast<ShortShared<kWarps>*>(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
  const int heads = p.kv_heads * chunks, s = blockIdx.x / heads, hv = blockIdx.x % heads;
  const int head = hv / chunks, first_q = hv % chunks * chunk_heads, columns = min(chunk_heads, p.group - first_q);
  if (!p.early) {
    pdl_wait();
    pdl_release();
  }
  const int length = tokens_of(p, s), held = (length + kBlock - 1) / kBlock;
  const int units = p.chosen == nullptr ? held : min(held, p.keep);
  // Chosen pages come from the preceding kernel, the tables do not.
  if (warp == 0) load_queries<kType, kE4m3>(p, sh.q, sh.to_log2, s, head * p.group + first_q, 0, columns, head);
  const auto stage_page = [&](int at, int logical, int page) {
    int valid = logical < 0 ? 0 : min(kBlock, length - logical * kBlock);
    if (logical >= 0 && (page < 0 || page >= p.pages)) {
      paged_error(p.status, kPagedBadPage);
      valid = 0;
    }
    sh.row[at] = (page * p.kv_heads + head) * kBlock;
    sh.valid[at] = valid;
  };
  const int32_t* table = p.tables + s * p.table_stride;
  if (warp == 1 && p.chosen == nullptr)
    for (int at = lane; at < units; at += 32) stage_page(at, at, table[at]);
  if (p.early) {
    pdl_wait();
    pdl_release();
  }
  if (warp == 1 && p.chosen != nullptr)
    for (int at = lane; at < units; at += 32) {
      int logical = p.chosen[(static_cast<long long>(s) * p.kv_heads + head) * p.keep + at];
      if (logical >= held) logical = -1;
      stage_page(at, logical, logical >= 0 ? table[logical] : -1);
    }
  __syncthreads();

  Running now;
  now.clear();
  const float2 to_log2 = *reinterpret_cast<const float2*>(&sh.to_log2[2 * j]);
  constexpr int kRowBytes = kDim * (kE4m3 ? 1 : 2), kChunks = kE4m3 ? 2 : 4, kHalves = kE4m3 ? 1 : 2;
  for (int at = warp; at < 4 * units; at += kWarps) {
    const int valid = sh.valid[at >> 2] - 16 * (at & 3);
    uint4 k[2][kChunks], v[4][kHalves];
    if (valid > 0) {
      const long long row = static_cast<long long>(sh.row[at >> 2] + 16 * (at & 3)) * kRowBytes;
      const auto load = [&](const void* rows, int key, int at16) {
        return key < valid ? load128(static_cast<const char*>(rows) + row + key * kRowBytes + at16 * 16) : make_uint4(0, 0, 0, 0);
      };
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) k[x][i] = load(p.k_cache, r + 8 * x, 8 * (i / 2) + 2 * j + i % 2);
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i][h] = load(p.v_cache, value_key(i, j), 8 * h + r);
    }
    if (valid > 0)
      attend_keys<kType, kE4m3>(
          now, to_log2, valid, [&](int i) { return sh.q[i][lane]; }, [&](int upper, int i) { return k[upper][i]; }, [] {}, [] {},
          [&](int i, int half) { return v[i][half]; });
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int d = 4; d < 32; d *= 2) now.l[c] += __shfl_xor_sync(~0u, now.l[c], d);
    if (r == 0) sh.m[warp][2 * j + c] = now.m[c], sh.l[warp][2 * j + c] = now.l[c];
    if (2 * j + c < columns && now.l[c] != 0.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sh.part[warp][c][i][lane] = make_float2(now.o[i][c], now.o[i][c + 2]);
    }
  }
  __syncthreads();
  if (threadIdx.x < 8 * kWarps) {
    const int col = threadIdx.x % 8, w = threadIdx.x / 8;
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) top = fmaxf(top, sh.m[x][col]);
    sh.f[w][col] = sh.l[w][col] == 0.f ? 0.f : exp2_fast(sh.m[w][col] - finite_or_zero(top));
    if (w == 0) sh.top[col] = top;
  }
  __syncthreads();
  const float v_scale = kE4m3 ? p.v_scale[head] : 1.f / kSmaller<kType, kE4m3>;
#pragma unroll
  for (int x = warp; x < 16; x += kWarps) {
    const int c = x / 8, i = x % 8, col = 2 * j + c, qh = head * p.group + first_q + col;
    if (col >= columns) continue;
    float sum = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = sh.f[w][col];
      sum += f * sh.l[w][col];
      if (f != 0.f) {  // a warp that saw no key has left nothing
        const float2 y = sh.part[w][c][i][lane];
        y0 += f * y.x, y1 += f * y.y;
      }
    }
    const float scale = sum == 0.f ? 0.f : v_scale / sum;
    store_pair<kType>(p, s, qh, dim_of<kE4m3>(i, r), y0 * scale, y1 * scale);
    if (i == 0 && r == 0 && p.lse != nullptr)
      p.lse[static_cast<long long>(s) * p.kv_heads * p.group + qh] = sum == 0.f ? -INFINITY : (sh.top[col] + log2f(sum)) * kLn2;
  }
}

template <int kType, bool kE4m3, int kWarps>
cudaError_t launch_warps(const PagedAttentionParams& p, int chunks, cudaStream_t stream) {
  const int chunk_heads = (p.group + chunks - 1) / chunks;
  return launch_overlapped<paged_short_attention_kernel<kType, kE4m3, kWarps>>(dim3(static_cast<unsigned>(p.requests) * p.kv_heads * chunks), 32 * kWarps,
                                                                             static_cast<int>(sizeof(ShortShared<kWarps>)), stream, p, chunks, chunk_heads);
}
// Warps of a CTA, for SMs of 16: few of them leave less to join, many shorten the chain of steps, and the last wave
// of CTAs should not be a small one.  128 tiles of 8 pages take 19.5, 12.8, 10.2 us with 4, 8, 16 warps, 512 tiles
// 29.7, 32.0, 36.6 us.
template <int kType, bool kE4m3>
cudaError_t launch_type(const PagedAttentionParams& p, int most_pages, cudaStream_t stream) {
  const int chunks = chunks_of(p.group);
  const int64_t tiles = static_cast<int64_t>(p.requests) * p.kv_heads * chunks;
  // Steps on an SM, one after the other: waves of CTAs, each of a warp's groups and what comes before and after.
  const auto steps = [&](int warps) {
    const int64_t waves = (tiles * warps + 148 * 16 - 1) / (148 * 16);
    return waves * ((4 * most_pages + warps - 1) / warps + 3);
  };
  if (steps(4) <= steps(8) && steps(4) <= steps(16)) return launch_warps<kType, kE4m3, 4>(p, chunks, stream);
  return steps(8) <= steps(16) ? launch_warps<kType, kE4m3, 8>(p, chunks, stream) : launch_warps<kType, kE4m3, 16>(p, chunks, stream);
}

}  // namespace

bool is_short_attention(int64_t tiles, int group, int most_pages, bool e4m3) {
  tiles *= chunks_of(group);
  // The split kernel's work is spread evenly, but costs more by tile (see the top).
  return most_pages <= (e4m3 ? (tiles < 32 ? 24 : kMostPages) : (tiles < 32 ? 12 : 16));
}

cudaError_t launch_paged_attention_short(const PagedAttentionParams& p, int most_pages, cudaStream_t stream) {
  const bool e4m3 = p.cache_dtype == kE4m3;
  if (p.dtype == kBf16) return e4m3 ? launch_type<kBf16, true>(p, most_pages, stream) : launch_type<kBf16, false>(p, most_pages, stream);
  return e4m3 ? launch_type<kFp16, true>(p, most_pages, stream) : launch_type<kFp16, false>(p, most_pages, stream);
}

}  // namespace vsa
