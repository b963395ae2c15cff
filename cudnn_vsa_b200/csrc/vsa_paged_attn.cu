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
//               programmatic stream serialisation, so that its launch latency is hidden.  Requests of few
//               pages have a kernel of their own (vsa_paged_attn_short.cu).
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
//   Rounding    Probabilities enter the second product as 16-bit terms that add up to them: three of BF16 (all 24
//               bits) or two of FP16 (an error of 2^-21).  One term would add an error as large as the output's own
//               rounding; two of BF16 (2^-15) left the decode layer over 720p contexts 2.6e-4 off FP32 arithmetic,
//               three leave 2.4e-5.  The third term costs what the loads do not hide: nothing at 113,648 tokens, 1 %
//               in full batches of 500 to 1,000 tokens, 2 to 8 % with 16 and 10 % with 32 query heads to a group.
//               All terms but the last are cut towards zero and none of a key that has weight is zero, so that an
//               infinite value is infinite in every product.  FP16 probabilities are scaled by 2^11 - up to 2^15 -
//               which puts the smallest FP16 number, the weight of a key that counts, at 2^-35 of the largest
//               probability; BF16 ones by 2^-32, so that sums of the largest values do not overflow, and a key has
//               weight from 2^-68 on.  For an e4m3 cache K, V and P are FP16 (every e4m3 value is one), and q is
//               scaled by a power of two per row so that FP16 holds it; e4m3 has no infinities, so both terms are
//               rounded to nearest. The second term costs there what it costs in instructions: the batch of 48 below
//               takes 181 us instead of 178, 207 instead of 192 on one GPU in a long run.
//
// Measured (one B200, 6.57 TB/s copy): 113,648 tokens x 12 heads in BF16, 698 MB, 108 us with the join
// (6.5 TB/s); 48 requests of up to 32,768 tokens in e4m3, seven heads a group, 1.14 GB, 181 us (6.3 TB/s; 193 to 207
// in a long run under the power cap); 32 ragged requests in FP16, 324 MB, 61 to 64 us (5.3 TB/s): of the 12 us above the
// bytes' time some 9 are the first lookups and loads, the last tile's products, and the join.
#include <cuda.h>

#include "vsa_kernels.h"
#include "vsa_paged_attn.cuh"

namespace vsa {

namespace {

constexpr int kWorkersMax = 160;  // one CTA per SM
constexpr int kJoinWarps = 8;

struct AttnParams {
  CUtensorMap k_map, v_map;
  PagedAttentionParams p;
  int chunks, chunk_heads;  // a group is taken in `chunks` parts of up to `chunk_heads` query heads
  float* partials;          // [2 * workers][chunk columns][128]
  float2* stats;            // [2 * workers][chunk columns] (maximum, sum)
  int4* split;              // [workers] {request, virtual head, last worker, 1} of the tile that starts here and goes on
};

VSA_DEVICE uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

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
  float m[kWarps][8], l[kWarps][8], f[kJoiners][kWarps][8];
  uint64_t full[2][kStages], empty[2][kStages];  // of K and V tiles
  uint64_t part_full, part_free, q_full[kTiles];
  int valid[kStages];
  int abort_flag;
};

template <int kType, bool kE4m3, int kC>
__global__ void __launch_bounds__(AttnShared<kE4m3, kC>::kThreads, 1) paged_attention_kernel(const __grid_constant__ AttnParams a) {
  using Shared = AttnShared<kE4m3, kC>;
  constexpr int kStages = Shared::kStages, kPages = Shared::kPages, kWarps = Shared::kWarps;
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
  // A short tile counts as kLeastTile pages: going from tile to tile costs a CTA some 3 us in its joining warps, however
  // few pages the tile has.  How many was tried out, not worked out (256 KiB are 5.9 us of an SM's share of HBM): ragged
  // requests of up to 40 pages, 320 tiles, 62 -> 45 us (e4m3, with one term of a probability, 54 -> 28).
  constexpr int kLeastTile = kE4m3 ? 16 : 8;
  const auto weight_of = [&](int units) { return units == 0 ? 0 : max(units, kLeastTile); };
  const WorkRange range = find_work([&](int s) { return weight_of(units_of(p, s)); }, p.requests, heads, worker, workers, 1, split);
  if (p.early) {
    pdl_wait();
    pdl_release();
  }
  __syncthreads();

  // The CTA's tiles, in order: every role walks them for itself.
  struct Walk {
    int s, hv, unit, left;  // the tile at hand, where this CTA enters it, the pages (as they count) left with it
    int count, end, last;   // its units, the first one that is not this CTA's, the same as they count
  };
  const auto leave = [&](Walk& w) {
    w.left -= w.last - w.unit;
    w.unit = 0;
    if (w.last == weight_of(w.count) && ++w.hv == heads) w.hv = 0, ++w.s;
  };
  const auto enter = [&](Walk& w) {  // false: no tile left
    while (w.left > 0) {
      while ((w.count = units_of(p, w.s)) == 0) ++w.s;
      w.last = min(weight_of(w.count), w.unit + w.left);
      w.end = min(w.last, w.count);
      if (w.unit < w.end) return true;
      leave(w);
    }
    return false;
  };
  Walk w{range.request, range.head, range.unit, range.end - range.begin, 0, 0, 0};
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
      x.n = min(32, w.end - base);
      x.head = w.hv / a.chunks;
      x.length = tokens_of(p, w.s);
      x.table = p.tables + w.s * p.table_stride;
      if (at < w.end) {
        x.logical = p.chosen == nullptr ? at : p.chosen[(static_cast<long long>(w.s) * p.kv_heads + x.head) * p.keep + at];
      }
      base += 32;
      if (base >= w.end) {
        leave(w);
        inside = enter(w);
        base = w.unit;
      }
      return x;
    };
    const auto look_up = [&](Piece& x) {
      if (x.logical >= (x.length + kBlock - 1) / kBlock) x.logical = -1;
      if (x.logical >= 0) x.page = x.table[x.logical];
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
      const int columns = min(a.chunk_heads, p.group - first_q);
#pragma unroll
      for (int t = 0; t < kC; ++t)
        load_queries<kType, kE4m3>(p, sh.q[buffer][t], &sh.to_log2[buffer][8 * t], w.s, head * p.group + first_q, 8 * t, columns, head);
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
    if (joiner == 0 && lane == 0) a.split[worker] = make_int4(0, 0, 0, 0);
    for (; enter(w); ++tiles_done, leave(w)) {
      const int s = w.s, head = w.hv / a.chunks, first_q = (w.hv % a.chunks) * a.chunk_heads, columns = min(a.chunk_heads, p.group - first_q);
      const bool starts = w.unit == 0, ends = w.end == w.count;
      mbar_wait(&sh.part_full, tiles_done & 1, &sh.abort_flag, p.status, 63);
      // The factors of the warps' results.  Lane: column `col` of the warps x + 4 k, whose column tile is k % kC.
      const int col = lane & 7, x = lane >> 3;
      const float out_scale = kE4m3 ? p.v_scale[head] : 1.f / kSmaller<kType, kE4m3>;
      float m[4], l[4], top[kC], sum[kC];
#pragma unroll
      for (int k = 0; k < 4; ++k) m[k] = sh.m[x + 4 * k][col], l[k] = sh.l[x + 4 * k][col];
#pragma unroll
      for (int t = 0; t < kC; ++t) {
        top[t] = m[t];
#pragma unroll
        for (int k = t + kC; k < 4; k += kC) top[t] = fmaxf(top[t], m[k]);
        top[t] = fmaxf(top[t], __shfl_xor_sync(~0u, top[t], 8));
        top[t] = fmaxf(top[t], __shfl_xor_sync(~0u, top[t], 16));
        sum[t] = 0.f;
#pragma unroll
        for (int k = t; k < 4; k += kC) {
          m[k] = l[k] == 0.f ? 0.f : exp2_fast(m[k] - finite_or_zero(top[t]));
          sum[t] += m[k] * l[k];
        }
        sum[t] += __shfl_xor_sync(~0u, sum[t], 8);
        sum[t] += __shfl_xor_sync(~0u, sum[t], 16);
        const float f = !(starts && ends) ? 1.f : sum[t] == 0.f ? 0.f : out_scale / sum[t];
#pragma unroll
        for (int k = t; k < 4; k += kC) sh.f[joiner][x + 4 * k][col] = m[k] * f;
        if (joiner == 0 && lane < 8 && 8 * t + col < columns) {
          const int qh = head * p.group + first_q + 8 * t + col;
          if (!(starts && ends)) a.stats[(2LL * worker + (starts ? 1 : 0)) * (8 * kC) + 8 * t + col] = make_float2(top[t], sum[t]);
          else if (p.lse != nullptr) p.lse[static_cast<long long>(s) * p.kv_heads * p.group + qh] = sum[t] == 0.f ? -INFINITY : (top[t] + log2f(sum[t])) * kLn2;
        }
      }
      __syncwarp();
      constexpr int kFrom = 4 * kPages;  // warps that hold a column tile
#pragma unroll
      for (int t = 0; t < kC; ++t) {
        const int first = 8 * t + 2 * j;  // this lane's columns: first, first + 1
        if (8 * t >= columns) break;
#pragma unroll
        for (int i = joiner; i < 8; i += Shared::kJoiners) {
          float2 y[2] = {};
#pragma unroll
          for (int z = 0; z < kFrom; ++z) {
            const int w = ((z / 4) * kC + t) * 4 + z % 4;
            const float2 f = *reinterpret_cast<const float2*>(&sh.f[joiner][w][2 * j]), v0 = sh.part[w][0][i][lane], v1 = sh.part[w][1][i][lane];
            y[0].x += f.x * v0.x, y[0].y += f.x * v0.y;
            y[1].x += f.y * v1.x, y[1].y += f.y * v1.y;
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (first + c >= columns) continue;
            const int d = dim_of<kE4m3>(i, r);
            if (starts && ends) store_pair<kType>(p, s, head * p.group + first_q + first + c, d, y[c].x, y[c].y);
            else *reinterpret_cast<float2*>(a.partials + ((2LL * worker + (starts ? 1 : 0)) * (8 * kC) + first + c) * kDim + d) = y[c];
          }
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
    Running now;
    now.clear();

    mbar_wait(&sh.q_full[tile], (tiles_done / Shared::kTiles) & 1, &sh.abort_flag, p.status, 65);
    const unsigned begin = g;
    const float2 to_log2 = *reinterpret_cast<const float2*>(&sh.to_log2[tile][8 * column_tile + 2 * j]);
    g += w.end - w.unit;
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
        attend_keys<kType, kE4m3>(
            now, to_log2, valid, [&](int i) { return sh.q[tile][column_tile][i][lane]; },
            [&](int upper, int i) { return lds128(k_tile + (i / 2) * kHalfTileBytes + 1024 * upper + r * 128 + (((2 * j + i % 2) ^ r) << 4)); },
            [&] {
              if (!Shared::kApart) return;
              __syncwarp();
              if (lane == 0) mbar_arrive(&sh.empty[0][stage]);
            },
            [&] {
              if (Shared::kApart) mbar_wait(&sh.full[1][stage], phase, &sh.abort_flag, p.status, 66);
            },
            [&](int i, int half) {
              const int key = value_key(i, j);
              return lds128(v_tile + half * kHalfTileBytes + key * 128 + ((r ^ (key & 7)) << 4));
            });
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[Shared::kApart ? 1 : 0][stage]);
    }

    // Leave the results to the joining warps and go on.
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int d = 4; d < 32; d *= 2) now.l[c] += __shfl_xor_sync(~0u, now.l[c], d);
    if (tiles_done > 0) mbar_wait(&sh.part_free, (tiles_done - 1) & 1, &sh.abort_flag, p.status, 62);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (r == 0) sh.m[warp][2 * j + c] = now.m[c], sh.l[warp][2 * j + c] = now.l[c];
      const bool some = now.l[c] != 0.f;  // without a key the products may be 0 * infinity
#pragma unroll
      for (int i = 0; i < 8; ++i) sh.part[warp][c][i][lane] = some ? make_float2(now.o[i][c], now.o[i][c + 2]) : make_float2(0.f, 0.f);
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
    const float f = sum == 0.f ? 0.f : (kE4m3 ? p.v_scale[head] : 1.f / kSmaller<kType, kE4m3>) / sum;
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
  if (err != cudaSuccess) return err;
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

int64_t paged_workspace_bytes(int64_t tiles, int group, int most_pages, bool e4m3) {
  if (is_short_attention(tiles, group, most_pages, e4m3)) return 0;
  const int64_t columns = columns_of(group);
  return kWorkersMax * (16 + 2 * columns * (kDim + 2) * static_cast<int64_t>(sizeof(float)));
}

int launch_paged_attention(const PagedAttentionParams& p, cudaStream_t stream) {
  const bool e4m3 = p.cache_dtype == kE4m3;
  const int most_pages = p.chosen == nullptr ? p.width : min(p.width, p.keep);
  if (is_short_attention(static_cast<int64_t>(p.requests) * p.kv_heads, p.group, most_pages, e4m3)) {
    const cudaError_t err = launch_paged_attention_short(p, most_pages, stream);
    return err == cudaSuccess ? kOk : kCudaError;
  }
  AttnParams a{};
  a.p = p;
  const long long rows = static_cast<long long>(p.pages) * p.kv_heads * kBlock;
  int rc = cache_map(&a.k_map, p.k_cache, rows, e4m3);
  if (rc == kOk) rc = cache_map(&a.v_map, p.v_cache, rows, e4m3);
  if (rc != kOk) return rc;
  const int columns = columns_of(p.group);
  a.chunks = (p.group + columns - 1) / columns;
  a.chunk_heads = (p.group + a.chunks - 1) / a.chunks;
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
