// Attention of one new token per request over its pages, or over the selected ones.
//
//   out_g = softmax(scale * q_g . K) V  [+ gate_g * coarse_g],   lse_g = log sum exp(scale * q_g . K)
//
// Every key and value byte is used for one product per query head of its group, so the kernel is
// bound by reading the cache from HBM: the design keeps those reads going without a pause.
//
//   Work split  All (request, key/value head, page) units are numbered in that order and every CTA
//               takes the same count of consecutive ones, whatever the lengths are.  The numbers
//               follow from `lengths` on the device: nothing is planned on the host.  A range covers
//               the end of one (request, head), whole ones, and the start of another; results of
//               incomplete ones go to the workspace as (maximum, sum, unnormalised output) and a
//               second small kernel joins them in the order of the workers.  It is launched with
//               programmatic stream serialisation, so that its launch latency is hidden.  Where no request can
//               have more than eight pages, CTAs take whole tiles and nothing is joined.
//   Loads       A warp looks the pages up (32 at a time) and fetches K and V tiles by TMA, 64 rows
//               of 256 bytes (16 bits) or 128 bytes (e4m3) with the 128-byte swizzle, into a ring
//               of 128 KiB: enough bytes in flight for an SM's share of HBM without occupancy.  Lookups run
//               three pieces ahead of the copies, and another warp stages the tiles' queries four tiles
//               ahead: a pause at each tile cost a batch of 48 ragged requests 5 %.
//   Products    S^T = K Q^T and O^T += V^T P^T on mma.m16n8k16: keys (then head dims) take the 16
//               rows and the group's query heads the 8 columns, so a group of eight wastes nothing;
//               tcgen05 would spend 64 rows on them, and the products are a tenth of the time of the
//               loads either way.  The order of the contraction index is free: lane (r, j) of a warp takes
//               16-byte chunks 2j and 2j+1 of key r, which feed the A operand as they are, and reads
//               all banks once under the swizzle.  For V^T two keys of one dim are paired by a byte
//               permute.  Four warps take 16 keys each of a page; four such groups take pages in turn
//               (the chain from the first product to the last is about 1500 cycles long, twice the time
//               a page takes to load), and with more than 8 or 16 query heads to a group two or four
//               of them take the same page, eight heads each.
//   Softmax     Running maximum per warp in base 2, raised only when a score exceeds it by 2^8 (2^4 with
//               FP16): the usual page costs one vote instead of a reduction.
//   Joining     The warps of a CTA leave their results of a tile in shared memory and go on with the
//               next; two warps of their own sum them up and write them.
//   Rounding    Probabilities enter the second product as two 16-bit terms (p = hi + lo, an error of
//               2^-15): one term would add an error as large as the output's own rounding.  hi is cut
//               towards zero and lo kept above zero, so that an infinite value is infinite in both
//               products.  FP16 probabilities are scaled by 2^11 - up to 2^15 - which puts the smallest
//               FP16 number at 2^-35 of the largest probability.  For an e4m3 cache K, V and P are FP16
//               (every e4m3 value is one), and q is scaled by a power of two per row so that FP16 holds
//               it; there one term's error of 2^-12 is small next to a BF16 output's 2^-9, and the
//               second term is left out for BF16 activations.
//
// Measured (one B200, 6.57 TB/s copy): 113,648 tokens x 12 heads in BF16, 698 MB, 108 us with the join
// (6.5 TB/s); 48 requests of up to 32,768 tokens in e4m3, seven heads a group, 1.14 GB, 179 us (6.4 TB/s); 32
// ragged requests in FP16, 324 MB, 64 us (5.1 TB/s): of the 14 us above the bytes' time some 9 are the
// first lookups and loads, the last tile's products, and the join.
#include <cuda.h>

#include "vsa_kernels.h"
#include "vsa_paged_common.cuh"

namespace vsa {

namespace {

constexpr int kWorkersMax = 160;  // one CTA per SM
constexpr int kJoinWarps = 8;
constexpr int kWholePages = 8;

struct AttnParams {
  CUtensorMap k_map, v_map;
  PagedAttentionParams p;
  int chunks, chunk_heads;  // a group is taken in `chunks` parts of up to `chunk_heads` query heads
  bool whole;               // tiles are not split
  float* partials;          // [2 * workers][chunk columns][128]
  float2* stats;            // [2 * workers][chunk columns] (maximum, sum)
  int4* split;              // [workers] {request, virtual head, last worker, 1} of the tile that starts here and goes on
};

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
VSA_DEVICE uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
VSA_DEVICE uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// 16-bit tiles: [half][row][128 bytes], one box; 8-bit tiles: [row][128 bytes].
template <bool kE4m3>
VSA_DEVICE void load_tile(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int row) {
  if (kE4m3)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(row) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(0) : "memory");
}

VSA_DEVICE int tokens_of(const PagedAttentionParams& p, int s) { return min(max(__ldg(p.lengths + s), 0), p.width * kBlock); }
// Units (pages) of every key/value head of request s.
VSA_DEVICE int units_of(const PagedAttentionParams& p, int s) {
  const int n = (tokens_of(p, s) + kBlock - 1) / kBlock;
  return p.chosen == nullptr ? n : min(n, p.keep);
}

// kC column tiles of eight query heads share a stage.
template <bool kE4m3, int kC>
struct AttnShared {
  static constexpr int kTile = kBlock * kDim * (kE4m3 ? 1 : 2);
  // Four groups of four warps: group g takes column tile g % kC of the pages whose number is
  // g / kC modulo kPages.
  static constexpr int kPages = 4 / kC, kWarps = 16, kJoiners = 2, kThreads = 32 * (kWarps + 2 + kJoiners);
  // A multiple of kPages, so that a stage always belongs to the same groups: they then wait for every
  // phase of its barriers and never for one that is two ahead.
  static constexpr int kStages = kE4m3 ? 8 : 4;
  static constexpr int kTiles = kC == 4 ? 2 : 4;  // tiles whose queries are staged
  // Whether K and V tiles have barriers of their own: a K tile is free after the first product then, and
  // K runs two units ahead of V.  16 bits gain 1 to 3 % (one request of 78,848 tokens: 57.5 -> 55.9 us).
  // 8-bit pages are bound by instructions, and the second wait and arrival of each warp cost them 10 %
  // (48 ragged requests: 181 -> 202 us).
  static constexpr bool kApart = !kE4m3;
  uint8_t tiles[kStages][2][kTile];
  uint4 q[kTiles][kC][4][32];     // Q^T fragments, per lane
  float to_log2[kTiles][8 * kC];  // factor of a query column's scores
  float2 part[kWarps][2][8][32];  // O^T fragments: column parity, product, lane
  float m[kWarps][8], l[kWarps][8];
  uint64_t full[2][kStages], empty[2][kStages];  // of K and V tiles
  uint64_t part_full, part_free, q_full[kTiles];
  int valid[kStages];
  int abort_flag;
};

// One warp: Q^T fragments of a tile.  Lane (r, j) holds query column r, its 16-byte chunks in the
// order in which the K operand takes them.
template <int kType, bool kE4m3, int kC, class Shared>
VSA_DEVICE void load_queries(const PagedAttentionParams& p, Shared& sh, int tile, int request, int first_head, int columns, int head) {
  const int lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
#pragma unroll
  for (int t = 0; t < kC; ++t) {
    const int col = 8 * t + r;
    const uint16_t* src = static_cast<const uint16_t*>(p.q) + request * p.q_row_stride +
                          static_cast<long long>(first_head + min(col, columns - 1)) * p.q_head_stride;
    uint32_t q[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // 16 bits: half i/2, chunk 2j + i%2, 8 dims.  8 bits: chunk 2j + i/2 of 16 dims, its half i%2.
      const int dim = kE4m3 ? 16 * (2 * j + i / 2) + 8 * (i % 2) : 64 * (i / 2) + 8 * (2 * j + i % 2);
      uint4 v = __ldg(reinterpret_cast<const uint4*>(src + dim));
      if (col >= columns) v = make_uint4(0, 0, 0, 0);
      q[4 * i] = v.x, q[4 * i + 1] = v.y, q[4 * i + 2] = v.z, q[4 * i + 3] = v.w;
    }
    float to_log2 = p.scale * kLog2e;
    if (kE4m3) {
      to_log2 *= __ldg(p.k_scale + head);
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
    for (int i = 0; i < 4; ++i) sh.q[tile][t][i][lane] = make_uint4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
    if (j == 0) sh.to_log2[tile][col] = to_log2;
  }
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

template <int kType, bool kE4m3, int kC>
__global__ void __launch_bounds__(AttnShared<kE4m3, kC>::kThreads, 1) paged_attention_kernel(const __grid_constant__ AttnParams a) {
  using Shared = AttnShared<kE4m3, kC>;
  constexpr int kStages = Shared::kStages, kPages = Shared::kPages, kWarps = Shared::kWarps;
  constexpr bool kHalf = kE4m3 || kType == kFp16;
  constexpr int kPType = kHalf ? kFp16 : kBf16;
  constexpr bool kTwoTerms = !kE4m3 || kType == kFp16;
  // `m` below is the running maximum less kShift, so that probabilities come out scaled by 2^kShift; it is
  // raised when a score exceeds it by kRaise.
  constexpr float kShift = kHalf ? 11.f : 0.f, kRaise = kHalf ? 15.f : 8.f;
  constexpr float kLeast = kHalf ? 5.9604644775390625e-8f : 1.17549435e-38f;  // smallest FP16; smallest normal BF16
  extern __shared__ uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw + ((1024 - (smem_u32(raw) & 1023)) & 1023));
  const PagedAttentionParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int worker = blockIdx.x, workers = gridDim.x, heads = p.kv_heads * a.chunks;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      for (int x = 0; x < 2; ++x) {
        mbar_init(&sh.full[x][i], 1);
        mbar_init(&sh.empty[x][i], 4 * kC);
      }
    }
    mbar_init(&sh.part_full, kWarps);
    mbar_init(&sh.part_free, Shared::kJoiners + 1);
    for (int i = 0; i < Shared::kTiles; ++i) mbar_init(&sh.q_full[i], 1);
    sh.abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == 32 * kWarps) tma_prefetch_desc(&a.k_map), tma_prefetch_desc(&a.v_map);
  if (!p.early) {
    pdl_wait();
    pdl_release();
  }
  WorkSplit split;
  // Shares of equal pages, or of whole tiles.
  const WorkRange range = find_work([&](int s) { return a.whole ? min(units_of(p, s), 1) : units_of(p, s); }, p.requests, heads, worker,
                                    workers, 1, split);
  if (p.early) {
    pdl_wait();
    pdl_release();
  }
  __syncthreads();

  // The CTA's tiles, in order: every role walks them for itself.
  struct Walk {
    int s, hv, unit, left;  // the tile at hand, the units (or whole tiles) left with it
    int count, last;        // its units, and the first one that is not this CTA's
  };
  const auto enter = [&](Walk& w) {  // false: no tile left
    if (w.left <= 0) return false;
    while ((w.count = units_of(p, w.s)) == 0) ++w.s;
    w.last = a.whole ? w.count : min(w.count, w.unit + w.left);
    return true;
  };
  const auto leave = [&](Walk& w) {
    w.left -= a.whole ? 1 : w.last - w.unit;
    w.unit = 0;
    if (w.last == w.count && ++w.hv == heads) w.hv = 0, ++w.s;
  };
  Walk w{range.request, range.head, range.unit, range.end - range.begin, 0, 0};
  unsigned tiles_done = 0;

  if (warp == kWarps) {
    // Loads.  Pieces of up to 32 units pass three stages: their logical pages are read two pieces ahead,
    // their physical pages one piece ahead.
    struct Piece {
      int n, head, length, logical, page;
      const int32_t* table;
    };
    bool inside = enter(w);
    int base = w.unit;
    const auto name = [&] {
      Piece x{0, 0, 0, -1, -1, nullptr};
      if (!inside) return x;
      const int at = base + lane;
      x.n = min(32, w.last - base);
      x.head = w.hv / a.chunks;
      x.length = tokens_of(p, w.s);
      x.table = p.tables + w.s * p.table_stride;
      if (at < w.last) {
        x.logical = p.chosen == nullptr ? at : p.chosen[(static_cast<long long>(w.s) * p.kv_heads + x.head) * p.keep + at];
      }
      base += 32;
      if (base >= w.last) {
        leave(w);
        inside = enter(w);
        base = w.unit;
      }
      return x;
    };
    const auto look_up = [&](Piece& x) {
      if (x.logical >= (x.length + kBlock - 1) / kBlock) x.logical = -1;
      if (x.logical >= 0) x.page = __ldg(x.table + x.logical);
    };
    // The tiles of unit g sit in stage g % kStages.
    unsigned g = 0;
    int rows[2] = {}, counts[2] = {};  // lane 0: units whose V tile is still to be fetched
    unsigned k_end = ~0u, v_end = ~0u;         // lane 0: the units that are not fetched, after a wait that gave up
    const auto fetch = [&](int which, unsigned unit, int row, int keys) {
      const int stage = unit % kStages;
      if (unit >= kStages && !mbar_wait(&sh.empty[which][stage], (unit / kStages - 1) & 1, &sh.abort_flag, p.status, 60))
        k_end = min(k_end, which == 0 ? unit : unit + 3), v_end = min(v_end, which == 1 ? unit : max(unit, 2u) - 2);
      if (unit >= (which == 0 ? k_end : v_end)) return;
      if (which == 0) sh.valid[stage] = keys;
      if (keys > 0) {
        mbar_expect_tx(&sh.full[which][stage], Shared::kApart ? Shared::kTile : 2 * Shared::kTile);
        load_tile<kE4m3>(smem_u32(sh.tiles[stage][which]), which == 0 ? &a.k_map : &a.v_map, &sh.full[which][stage], row);
        if (!Shared::kApart) load_tile<kE4m3>(smem_u32(sh.tiles[stage][1]), &a.v_map, &sh.full[0][stage], row);
      } else {
        mbar_arrive(&sh.full[which][stage]);
      }
    };
    Piece now = name();
    Piece next = name();
    look_up(now);
    while (now.n > 0) {
      const Piece after = name();
      look_up(next);
      int valid = now.logical < 0 ? 0 : min(kBlock, now.length - now.logical * kBlock);
      if (now.logical >= 0 && (now.page < 0 || now.page >= p.pages)) {
        paged_error(p.status, kPagedBadPage);
        valid = 0;
      }
      const int row = (now.page * p.kv_heads + now.head) * kBlock;
      for (int i = 0; i < now.n; ++i, ++g) {
        const int keys = __shfl_sync(~0u, valid, i), first = __shfl_sync(~0u, row, i);
        if (lane == 0) {
          fetch(0, g, first, keys);
          if (Shared::kApart) {
            if (g >= 2) fetch(1, g - 2, rows[0], counts[0]);
            rows[0] = rows[1], counts[0] = counts[1];
            rows[1] = first, counts[1] = keys;
          }
        }
      }
      now = next;
      next = after;
    }
    if (lane == 0) {
      if (Shared::kApart && g >= 2) fetch(1, g - 2, rows[0], counts[0]);
      if (Shared::kApart && g >= 1) fetch(1, g - 1, rows[1], counts[1]);
      // No copy is in flight when the CTA ends, not even after a wait that gave up.
      int heedless = 0;
      const auto landed = [&](uint64_t* full, unsigned end) {
        for (unsigned u = max(end, static_cast<unsigned>(kStages)) - kStages; u < end; ++u)
          mbar_wait(&full[u % kStages], (u / kStages) & 1, &heedless, p.status, 67);
      };
      landed(sh.full[0], min(g, k_end));
      if (Shared::kApart) landed(sh.full[1], min(g, v_end));
    }
    return;
  }

  if (warp == kWarps + 1) {
    // Queries: kTiles tiles ahead of the one that the other warps have finished.
    const auto stage_queries = [&](int buffer) {
      const int head = w.hv / a.chunks, first_q = (w.hv % a.chunks) * a.chunk_heads;
      load_queries<kType, kE4m3, kC>(p, sh, buffer, w.s, head * p.group + first_q, min(a.chunk_heads, p.group - first_q), head);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full[buffer]);
      leave(w);
    };
    unsigned staged = 0;
    while (staged < Shared::kTiles && enter(w)) stage_queries(staged++);
    for (; tiles_done < staged; ++tiles_done) {
      mbar_wait(&sh.part_full, tiles_done & 1, &sh.abort_flag, p.status, 64);
      if (lane == 0) mbar_arrive(&sh.part_free);
      if (enter(w)) stage_queries(staged++ % Shared::kTiles);
    }
    return;
  }

  if (warp > kWarps + 1) {
    const int joiner = warp - kWarps - 2, r = lane >> 2, j = lane & 3;
    if (joiner == 0 && lane == 0 && !a.whole) a.split[worker] = make_int4(0, 0, 0, 0);
    for (; enter(w); ++tiles_done, leave(w)) {
      const int s = w.s, head = w.hv / a.chunks, first_q = (w.hv % a.chunks) * a.chunk_heads, columns = min(a.chunk_heads, p.group - first_q);
      const bool starts = w.unit == 0, ends = w.last == w.count;
      mbar_wait(&sh.part_full, tiles_done & 1, &sh.abort_flag, p.status, 63);
      constexpr int kFrom = 4 * kPages;  // warps that hold a column tile
#pragma unroll
      for (int t = 0; t < kC; ++t)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = 8 * t + 2 * j + c, qh = head * p.group + first_q + col;
          if (col >= columns) continue;
          const auto from = [&](int x) { return ((x / 4) * kC + t) * 4 + x % 4; };
          float top = -INFINITY, sum = 0.f, f[kFrom];
#pragma unroll
          for (int x = 0; x < kFrom; ++x) top = fmaxf(top, sh.m[from(x)][2 * j + c]);
#pragma unroll
          for (int x = 0; x < kFrom; ++x) {
            const float l = sh.l[from(x)][2 * j + c];
            f[x] = l == 0.f ? 0.f : exp2_fast(sh.m[from(x)][2 * j + c] - finite_or_zero(top));
            sum += f[x] * l;
          }
          const float scale = sum == 0.f ? 0.f : (kE4m3 ? __ldg(p.v_scale + head) : 1.f) / sum;
          const long long slot = (2LL * worker + (starts ? 1 : 0)) * (8 * kC) + col;
          for (int i = joiner; i < 8; i += Shared::kJoiners) {
            float y0 = 0.f, y1 = 0.f;
#pragma unroll
            for (int x = 0; x < kFrom; ++x)
              if (f[x] != 0.f) {  // a warp that saw no key has left nothing
                const float2 v = sh.part[from(x)][c][i][lane];
                y0 += f[x] * v.x, y1 += f[x] * v.y;
              }
            const int d = kE4m3 ? 16 * r + 2 * i : 64 * (i / 4) + 8 * r + 2 * (i % 4);
            if (starts && ends) store_pair<kType>(p, s, qh, d, y0 * scale, y1 * scale);
            else *reinterpret_cast<float2*>(a.partials + slot * kDim + d) = make_float2(y0, y1);
          }
          if (joiner == 0 && r == 0) {
            if (!(starts && ends)) a.stats[slot] = make_float2(top, sum);
            else if (p.lse != nullptr) p.lse[static_cast<long long>(s) * p.kv_heads * p.group + qh] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
          }
        }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh.part_free);
        if (joiner == 0 && starts && !ends) a.split[worker] = make_int4(s, w.hv, split.owner(range.end + (w.count - w.last) - 1), 1);
      }
    }
    // Requests without tokens have no units.
    for (int e = worker; e < p.requests; e += workers) {
      if (units_of(p, e) > 0) continue;
      for (int qh = joiner; qh < p.kv_heads * p.group; qh += Shared::kJoiners) {
        store_pair<kType>(p, e, qh, 4 * lane, 0.f, 0.f);
        store_pair<kType>(p, e, qh, 4 * lane + 2, 0.f, 0.f);
        if (p.lse != nullptr && lane == 0) p.lse[static_cast<long long>(e) * p.kv_heads * p.group + qh] = -INFINITY;
      }
    }
    return;
  }

  const int r = lane >> 2, j = lane & 3, column_tile = (warp >> 2) % kC, turn = (warp >> 2) / kC, row0 = (warp & 3) * 16;
  unsigned g = 0;
  for (; enter(w); leave(w)) {
    const int first_q = (w.hv % a.chunks) * a.chunk_heads, columns = min(a.chunk_heads, p.group - first_q), tile = tiles_done % Shared::kTiles;
    float o[8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    mbar_wait(&sh.q_full[tile], (tiles_done / Shared::kTiles) & 1, &sh.abort_flag, p.status, 65);
    const unsigned begin = g;
    const float2 to_log2 = *reinterpret_cast<const float2*>(&sh.to_log2[tile][8 * column_tile + 2 * j]);
    // `base` is the running maximum, or 0 as long as it is -infinity; a score (less base) above `limit` raises it.
    float base[2] = {}, limit[2] = {-INFINITY, -INFINITY};
    g += w.last - w.unit;
    for (unsigned u = begin + (static_cast<unsigned>(turn) - begin) % kPages; u < g; u += kPages) {
      const int stage = u % kStages;
      const uint32_t phase = (u / kStages) & 1;
      mbar_wait(&sh.full[0][stage], phase, &sh.abort_flag, p.status, 61);
      const int valid = sh.valid[stage] - row0;  // of this warp's 16 keys
      if (valid <= 0) {
        if (Shared::kApart) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.empty[0][stage]);
          mbar_wait(&sh.full[1][stage], phase, &sh.abort_flag, p.status, 66);
        }
      } else {
        const uint32_t k_tile = smem_u32(sh.tiles[stage][0]) + row0 * 128, v_tile = smem_u32(sh.tiles[stage][1]) + row0 * 128;
        float acc[2][4] = {};
        if (kE4m3) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t at16 = r * 128 + (((2 * j + i) ^ r) << 4);
            const uint4 q[2] = {sh.q[tile][column_tile][2 * i][lane], sh.q[tile][column_tile][2 * i + 1][lane]};
            const uint4 x = lds128(k_tile + at16), y = lds128(k_tile + 1024 + at16);
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
            const uint32_t at16 = (i / 2) * kHalfTileBytes + r * 128 + (((2 * j + i % 2) ^ r) << 4);
            const uint4 x = lds128(k_tile + at16), y = lds128(k_tile + 1024 + at16);
            const uint4 q = sh.q[tile][column_tile][i][lane];
            mma16816<kHalf>(acc[0], x.x, y.x, x.y, y.y, q.x, q.y);
            mma16816<kHalf>(acc[1], x.z, y.z, x.w, y.w, q.z, q.w);
          }
        }
        if (Shared::kApart) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.empty[0][stage]);
        }
        // Scores in base 2, less `base`: rows are keys r and r + 8, columns query heads 2j and 2j + 1.
        float sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[0][i] += acc[1][i];
          sc[i] = fmaf(acc[0][i], (i & 1) ? to_log2.y : to_log2.x, -base[i & 1]);
        }
        if (valid < 16) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (r + 8 * (i / 2) >= valid) sc[i] = -INFINITY;
        }
        if (__any_sync(~0u, fmaxf(sc[0], sc[2]) > limit[0] || fmaxf(sc[1], sc[3]) > limit[1])) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = fmaxf(sc[c], sc[c + 2]);
#pragma unroll
            for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
            top = fmaxf(m[c], top + base[c] - kShift);
            const float now = finite_or_zero(top), shrink = exp2_fast(m[c] - now);
#pragma unroll
            for (int i = c; i < 4; i += 2)
              if (sc[i] != -INFINITY) sc[i] = fmaf(acc[0][i], (i & 1) ? to_log2.y : to_log2.x, -now);
            m[c] = top, base[c] = now;
            if (top != -INFINITY) limit[c] = kRaise;
            l[c] *= shrink;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i][c] *= shrink, o[i][c + 2] *= shrink;
          }
        }
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float p0 = exp2_fast(sc[2 * x]), p1 = exp2_fast(sc[2 * x + 1]);
          l[0] += p0;
          l[1] += p1;
          if (kTwoTerms) {
            if (kHalf) p0 = fmaxf(p0, kLeast), p1 = fmaxf(p1, kLeast);
            const uint32_t both = truncate2<kHalf>(p0, p1);
            const float h0 = unpack1<kPType>(both & 0xFFFF), h1 = unpack1<kPType>(both >> 16);
            hi[x] = transpose8x8(both);
            lo[x] = transpose8x8(pack2<kPType>(fmaxf(p0 - h0, kLeast), fmaxf(p1 - h1, kLeast)));
          } else {
            hi[x] = transpose8x8(pack2<kPType>(p0, p1));
          }
        }
        if (Shared::kApart) mbar_wait(&sh.full[1][stage], phase, &sh.abort_flag, p.status, 66);
        // V^T: rows are dims, columns keys; this lane's keys are 2j, 2j+1, 2j+8, 2j+9.
        const auto clear_rows = [&](uint4 (&v)[4]) {  // what is behind the request's last token
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (2 * j + (i & 1) + 8 * (i >> 1) >= valid) v[i] = make_uint4(0, 0, 0, 0);
        };
        if (kE4m3) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 2 * j + (i & 1) + 8 * (i >> 1);
            v[i] = lds128(v_tile + key * 128 + ((r ^ (key & 7)) << 4));
          }
          if (valid < 16) clear_rows(v);
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // rows r: dim 16 r + 2 i, rows r + 8: dim 16 r + 2 i + 1
            const uint32_t pick = (i & 1) ? 0x7362u : 0x5140u;
            const uint32_t x = __byte_perm(word(v[0], i / 2), word(v[1], i / 2), pick);
            const uint32_t y = __byte_perm(word(v[2], i / 2), word(v[3], i / 2), pick);
            const uint32_t a0 = e4m3x2_to_half2(x & 0xFFFF), a1 = e4m3x2_to_half2(x >> 16);
            const uint32_t a2 = e4m3x2_to_half2(y & 0xFFFF), a3 = e4m3x2_to_half2(y >> 16);
            mma16816<true>(o[i], a0, a1, a2, a3, hi[0], hi[1]);
            if (kTwoTerms) mma16816<true>(o[i], a0, a1, a2, a3, lo[0], lo[1]);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = 2 * j + (i & 1) + 8 * (i >> 1);
              v[i] = lds128(v_tile + h * kHalfTileBytes + key * 128 + ((r ^ (key & 7)) << 4));
            }
            if (valid < 16) clear_rows(v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // rows r: dim 64 h + 8 r + 2 e, rows r + 8: the next dim
              const uint32_t a0 = __byte_perm(word(v[0], e), word(v[1], e), 0x5410u), a1 = __byte_perm(word(v[0], e), word(v[1], e), 0x7632u);
              const uint32_t a2 = __byte_perm(word(v[2], e), word(v[3], e), 0x5410u), a3 = __byte_perm(word(v[2], e), word(v[3], e), 0x7632u);
              mma16816<kHalf>(o[4 * h + e], a0, a1, a2, a3, hi[0], hi[1]);
              if (kTwoTerms) mma16816<kHalf>(o[4 * h + e], a0, a1, a2, a3, lo[0], lo[1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[Shared::kApart ? 1 : 0][stage]);
    }

    // Leave the results to the joining warps and go on.
    if (tiles_done > 0) mbar_wait(&sh.part_free, (tiles_done - 1) & 1, &sh.abort_flag, p.status, 62);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int d = 4; d < 32; d *= 2) l[c] += __shfl_xor_sync(~0u, l[c], d);
      if (r == 0) sh.m[warp][2 * j + c] = m[c], sh.l[warp][2 * j + c] = l[c];
      if (8 * column_tile + 2 * j + c < columns && l[c] != 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sh.part[warp][c][i][lane] = make_float2(o[i][c], o[i][c + 2]);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.part_full);
    ++tiles_done;
  }
}

// Joins the partial results of the tile that starts in worker blockIdx.x and goes on behind it: every
// gridDim.y-th query head from blockIdx.y on.
template <int kType, bool kE4m3>
__global__ void __launch_bounds__(32 * kJoinWarps, 4) paged_join_kernel(const __grid_constant__ AttnParams a, int slots) {
  __shared__ __align__(16) float4 part[kJoinWarps][32];
  pdl_wait();
  pdl_release();
  const PagedAttentionParams& p = a.p;
  const int4 tile = a.split[blockIdx.x];
  if (tile.w == 0) return;
  const int head = tile.y / a.chunks, first_q = (tile.y % a.chunks) * a.chunk_heads, lane = threadIdx.x & 31;
  const int columns = min(a.chunk_heads, p.group - first_q);
  for (int column = blockIdx.y; column < columns; column += gridDim.y)
    join_partials<kJoinWarps>(threadIdx.x >> 5, 1, blockIdx.x, tile.z, column, column + 1, slots, a.stats, a.partials, part, [&](int col, float top, float sum, float4 y) {
    const float f = sum == 0.f ? 0.f : (kE4m3 ? __ldg(p.v_scale + head) : 1.f) / sum;
    const int qh = head * p.group + first_q + col;
    if (sum == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
    store_pair<kType>(p, tile.x, qh, 4 * lane, y.x * f, y.y * f);
    store_pair<kType>(p, tile.x, qh, 4 * lane + 2, y.z * f, y.w * f);
    if (p.lse != nullptr && lane == 0)
      p.lse[static_cast<long long>(tile.x) * p.kv_heads * p.group + qh] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  });
}

// [pages * kv_heads * 64] rows of 128 values as boxes of 64 rows.
int cache_map(CUtensorMap* map, const void* base, long long rows, bool e4m3) {
  const TensorMapEncoder encode = tensor_map_encoder();
  if (encode == nullptr) return kNoDriverEntry;
  const cuuint32_t ones[3] = {1, 1, 1};
  CUresult res;
  if (e4m3) {
    const cuuint64_t dims[2] = {kDim, static_cast<cuuint64_t>(rows)}, strides[1] = {kDim};
    const cuuint32_t box[2] = {kDim, kBlock};
    res = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    const cuuint64_t dims[3] = {64, static_cast<cuuint64_t>(rows), 2}, strides[2] = {2 * kDim, 128};
    const cuuint32_t box[3] = {64, kBlock, 2};
    res = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  return res == CUDA_SUCCESS ? kOk : kTensorMapError;
}

template <int kType, bool kE4m3, int kC>
cudaError_t launch(const AttnParams& a, int workers, cudaStream_t stream) {
  const int smem = static_cast<int>(sizeof(AttnShared<kE4m3, kC>)) + 1024;
  static_assert(sizeof(AttnShared<kE4m3, kC>) + 1024 <= 227 * 1024, "shared memory of one CTA");
  const cudaError_t err = launch_overlapped<paged_attention_kernel<kType, kE4m3, kC>>(dim3(workers), AttnShared<kE4m3, kC>::kThreads, smem, stream, a);
  if (err != cudaSuccess || a.whole) return err;
  return launch_overlapped<paged_join_kernel<kType, kE4m3>>(dim3(workers, a.chunk_heads < 4 ? a.chunk_heads : 4), 32 * kJoinWarps, 0, stream, a, 8 * kC);
}

template <int kType, bool kE4m3>
cudaError_t launch_columns(const AttnParams& a, int columns, int workers, cudaStream_t stream) {
  if (columns == 8) return launch<kType, kE4m3, 1>(a, workers, stream);
  if (columns == 16) return launch<kType, kE4m3, 2>(a, workers, stream);
  return launch<kType, kE4m3, 4>(a, workers, stream);
}

// Query columns that share a pass over the keys: what holds the group, 32 at most.
int columns_of(int group) { return group <= 8 ? 8 : group <= 16 ? 16 : 32; }

}  // namespace

int64_t paged_workspace_bytes(int group, int most_pages) {
  if (most_pages <= kWholePages) return 0;
  const int64_t columns = columns_of(group);
  return kWorkersMax * (16 + 2 * columns * (kDim + 2) * static_cast<int64_t>(sizeof(float)));
}

int launch_paged_attention(const PagedAttentionParams& p, cudaStream_t stream) {
  AttnParams a{};
  a.p = p;
  const bool e4m3 = p.cache_dtype == kE4m3;
  const long long rows = static_cast<long long>(p.pages) * p.kv_heads * kBlock;
  int rc = cache_map(&a.k_map, p.k_cache, rows, e4m3);
  if (rc == kOk) rc = cache_map(&a.v_map, p.v_cache, rows, e4m3);
  if (rc != kOk) return rc;
  const int columns = columns_of(p.group);
  a.chunks = (p.group + columns - 1) / columns;
  a.chunk_heads = (p.group + a.chunks - 1) / a.chunks;
  // Tiles of at most eight pages - two rounds of the four groups of warps - are not worth a second
  // kernel: one request of 100 tokens takes 9.1 us in two kernels.
  a.whole = (p.chosen == nullptr ? p.width : min(p.width, p.keep)) <= kWholePages;
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return kCudaError;
  const int workers = sms < kWorkersMax ? sms : kWorkersMax;
  char* at = reinterpret_cast<char*>(p.workspace);
  a.split = reinterpret_cast<int4*>(at);
  a.stats = reinterpret_cast<float2*>(at + kWorkersMax * 16);
  a.partials = reinterpret_cast<float*>(at + kWorkersMax * (16 + 2 * columns * 8));
  cudaError_t err;
  if (p.dtype == kBf16) err = e4m3 ? launch_columns<kBf16, true>(a, columns, workers, stream) : launch_columns<kBf16, false>(a, columns, workers, stream);
  else err = e4m3 ? launch_columns<kFp16, true>(a, columns, workers, stream) : launch_columns<kFp16, false>(a, columns, workers, stream);
  return err == cudaSuccess ? kOk : kCudaError;
}

}  // namespace vsa
