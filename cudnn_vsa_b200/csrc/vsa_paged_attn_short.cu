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
// Time against the split kernel, us (this kernel : the split one), BF16 with 4 query heads to a key/value head, e4m3
// with 8; tiles of equal and of ragged length:
//    tiles pages       equal, BF16      ragged, BF16       equal, e4m3      ragged, e4m3
//        8     8      7.6 :   9.7      7.6 :   9.7      5.9 :  10.0      5.8 :   9.9
//        8    12      9.6 :   9.8      9.5 :   9.7      6.8 :  10.2      7.0 :  10.3
//        8    16     11.5 :  10.0     11.5 :  10.0      8.0 :  10.8      8.0 :  10.7
//        8    24     15.3 :  10.0     15.3 :  10.0     10.0 :  11.0     10.0 :  10.9
//        8    32     19.0 :  10.3     19.1 :  10.2     12.1 :  11.1     12.0 :  11.2
//       80     8      8.4 :  13.9      7.6 :  13.3      6.2 :  13.8      6.0 :  12.5
//       80    12     11.5 :  16.8      9.6 :  13.9      7.4 :  15.0      7.1 :  14.3
//       80    16     13.6 :  18.3     11.8 :  14.4      8.7 :  16.2      8.0 :  15.4
//       80    24     17.9 :  21.2     16.8 :  16.4     12.5 :  18.7     10.3 :  16.0
//       80    32     22.2 :  24.0     21.2 :  18.2     15.0 :  20.1     12.9 :  16.6
//      320     8     22.8 :  25.2     19.6 :  22.6     14.8 :  21.6     11.5 :  19.2
//      320    12     31.9 :  31.6     26.9 :  24.8     19.7 :  24.5     16.6 :  22.9
//      320    16     40.6 :  38.8     34.0 :  27.0     24.7 :  28.6     20.7 :  26.5
//      320    24     58.2 :  49.6     48.8 :  33.3     34.4 :  33.5     28.3 :  28.3
//      320    32     69.1 :  62.3     38.1 :  39.7     42.7 :  41.2     25.4 :  30.5
//    1,600     8     72.4 :  76.2     43.9 :  62.2     44.0 :  52.7     28.6 :  49.2
//    1,600    12    102.8 : 106.0     60.4 :  71.2     60.1 :  66.4     38.0 :  62.1
//    1,600    16    133.5 : 136.2     77.2 :  82.1     76.3 :  81.3     46.3 :  75.5
//    1,600    24    194.6 : 195.8    111.7 : 108.4    108.4 : 111.7     63.9 :  81.1
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
  // The split kernel's work is spread evenly, but costs more by tile.  The limits are where the table at the top changes
  // sides for few tiles, and for all numbers of tiles from 32 on taken together.  With one number for these the rule is
  // off in places: 320 BF16 tiles of 16 pages would be faster split (equal 4 %, ragged 20 %; of 12 pages ragged 8 %), 80
  // BF16 tiles of 24 and 32 pages faster unsplit (16 and 8 %), 320 e4m3 tiles of 24 and 32 pages faster split (3 %).
  return most_pages <= (e4m3 ? (tiles < 32 ? 24 : kMostPages) : (tiles < 32 ? 12 : 16));
}

cudaError_t launch_paged_attention_short(const PagedAttentionParams& p, int most_pages, cudaStream_t stream) {
  const bool e4m3 = p.cache_dtype == kE4m3;
  if (p.dtype == kBf16) return e4m3 ? launch_type<kBf16, true>(p, most_pages, stream) : launch_type<kBf16, false>(p, most_pages, stream);
  return e4m3 ? launch_type<kFp16, true>(p, most_pages, stream) : launch_type<kFp16, false>(p, most_pages, stream);
}

}  // namespace vsa
