// Append, selection and compaction of a paged 16-bit cache that evicts tokens by their
// accumulated attention weight. No reference counterpart.
//
// A token's state is kept by (sequence, kv head, logical slot): scores [B, H, T] fp32 and
// positions [B, H, T] int32, where T covers the slots of a sequence. Attention does not depend
// on the order of the cached tokens, so an eviction need not keep it: the kept tokens of the
// slots >= budget (movers) go into the evicted slots < budget (holes), and everything else
// stays where it is. Sources (>= budget) and destinations (< budget) are disjoint, so
// the rows move in place, in any order, and a second run of the same moves changes nothing.
// A page past the budget costs a few rows this way, where keeping the order would move half
// of the cache. Positions say which tokens are the newest, since slots no longer do.
#include <cooperative_groups.h>

#include "common.cuh"
#include "decode_common.h"

namespace cg = cooperative_groups;

namespace bpt {
namespace {

// ------------------------------------------------------------------------------- selection
//
// The budget-th largest key of a row is found by a radix select over the scores' bits, mapped
// to unsigned keys of the same order: passes over 11 + 11 + 10 bits, each a histogram of the
// keys that share the digits found so far, and no further pass once a bin is taken whole. One
// cluster of C CTAs takes one (sequence, kv head). Each CTA reads its slice of the scores and
// positions once and keeps the keys in registers (TILES of 4 a thread; longer slices are read
// again in each pass); histograms and prefix counts are exchanged through distributed shared
// memory. Ties at the threshold go to the lowest slots, so the result is unique and does not
// depend on the order in which the histogram's integer atomics arrive.
//
// 8 bytes a slot would take 1.3 to 2.2 us in the cases below; what bounds the kernel is a chain
// of latencies: lengths, keys (1.7 us together), and per pass a histogram and its scan (1 us in
// one CTA, 2.5 to 3 us across a cluster). Measured: B=32 x 8 heads of 4112 slots 7.0 us (one CTA
// a row; 10.0 when the zero scores shared a bin and took all three passes), 8 heads of 128k slots
// 14.7 us (clusters of 16; 15.4 with 8), B=8 x 8 heads of 16-32k slots 14.7 us (clusters of 4; 16.4
// with 2). The simple form, keys in shared memory and three passes always, took 18.8, 36.7 and
// 30.7 us.

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kGroups = kBins / 128;         // a lane's 4 bins times a warp
constexpr int kTile = 128;                   // slots that a warp takes at a time, 4 a lane
constexpr int kMaxTiles = 16;                // tiles of a warp that stay in registers
constexpr int kMaxCluster = 16;                // above 8: not portable, B200 has them
constexpr uint32_t kProtectedKey = 0xffffffffu;
constexpr uint32_t kBinKeys = 1u << 21;      // keys of one bin of the first pass
constexpr uint32_t kZeroBin = 1024u, kProtectedBin = 2047u;
constexpr uint32_t kNoKey = 0u;              // past the end; a score's key is at least 1

struct SelectParams {
  const float* scores;
  int64_t sc_sb, sc_sh;
  const int32_t* positions;
  int64_t pos_sb, pos_sh;
  const int32_t* seq_lens;
  const int32_t* next_pos;
  int kv_heads, slots, budget, recent, sinks;
  int32_t *src, *dst;                        // [B, H, moves]
  int moves;
  int32_t* counts;                           // [B, H]
  int32_t* new_lens;                         // [B]
  int vec;                                   // rows are 16-byte aligned
};

// Unsigned key of the same order as the score: NaN lowest, -0 equal to +0. Positive scores are
// one bin of the first pass higher than their bits, so that 0, the score of new tokens and of
// weights that underflow, has a bin for itself and a threshold there needs no further pass.
__device__ __forceinline__ uint32_t score_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  if (f != f) return 1u;
  if (u & 0x80000000u) return ~u;
  return u + (u ? 0x80000000u + kBinKeys : 0x80000000u);
}

__device__ __forceinline__ uint32_t warp_inclusive(uint32_t x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(kFullMask, x, o);
    if (lane >= o) x += up;
  }
  return x;
}

// Sum of v[0 .. i), i <= 32.
__device__ __forceinline__ uint32_t sum_below(const uint32_t* v, int i, int lane) {
  return __reduce_add_sync(kFullMask, lane < i ? v[lane] : 0u);
}

template <int TILES>
__global__ void __launch_bounds__(kSelThreads, TILES <= 4 ? 2 : 1)
select_kernel(const SelectParams p) {
  static_assert(kSelWarps <= 32, "one lane per warp in the block-wide sums");
  static_assert(kBins == 4 * kSelThreads && kGroups == kSelWarps, "4 bins a thread");
  static_assert(kMaxCluster <= kSelWarps, "one warp per CTA of the cluster");
  // a histogram and, past it, one bin that nobody reads for the slots past the end
  __shared__ __align__(16) uint32_t s_hist[2][kBins + 4];
  __shared__ uint32_t s_group[2][kGroups];   // sums of 128 bins, from the top
  // C > 1: the CTAs' group sums, and their bins of the group that is searched
  __shared__ uint32_t s_groups[kMaxCluster][kGroups];
  __shared__ __align__(16) uint4 s_bins[kMaxCluster][32];
  __shared__ uint32_t s_rank_gt[kMaxCluster], s_rank_eq[kMaxCluster];
  __shared__ uint32_t s_digit, s_left, s_bin;
  __shared__ uint32_t s_gt[kSelWarps], s_eq[kSelWarps];

  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = int(blockIdx.x) / C;
  const int b = row / p.kv_heads, h = row % p.kv_heads;

#pragma unroll
  for (int i = 0; i < 2; ++i)
    *reinterpret_cast<uint4*>(&s_hist[i][4 * tid]) = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int n = min(max(p.seq_lens[b], 0), p.slots);
  // 64-bit: next_pos - recent may pass the int range
  const int64_t first_recent = int64_t(p.next_pos[b]) - p.recent;
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = min(n, p.budget);
  int32_t* src = p.src + int64_t(row) * p.moves;
  int32_t* dst = p.dst + int64_t(row) * p.moves;
  // unused places; the barriers of the passes order this before the moves of any CTA
  for (int i = rank * kSelThreads + tid; i < p.moves; i += C * kSelThreads) {
    src[i] = -1;
    dst[i] = -1;
  }
  if (n <= p.budget) {                       // the same n in every CTA of the cluster
    if (rank == 0 && tid == 0) p.counts[row] = 0;
    return;
  }

  // this CTA's slots, and this warp's [w_lo, w_hi) of them: whole tiles
  const int per = cdiv(cdiv(n, C), kTile) * kTile;
  const int lo = min(n, rank * per), hi = min(n, lo + per);
  const int w_per = cdiv(cdiv(per, kSelWarps), kTile) * kTile;
  const int w_lo = min(hi, lo + warp * w_per), w_hi = min(hi, w_lo + w_per);
  const float* sc = p.scores + int64_t(b) * p.sc_sb + int64_t(h) * p.sc_sh;
  const int32_t* pos = p.positions + int64_t(b) * p.pos_sb + int64_t(h) * p.pos_sh;
  const int32_t sinks = p.sinks;
  auto key_of = [&](float f, int32_t at) {
    return (at < sinks || at >= first_recent) ? kProtectedKey : score_key(f);
  };
  // keys of slots i .. i + 3 of the row
  auto read4 = [&](int i, uint32_t (&k)[4]) {
    if (p.vec && i + 4 <= w_hi) {
      const float4 f = *reinterpret_cast<const float4*>(sc + i);
      const int4 at = *reinterpret_cast<const int4*>(pos + i);
      k[0] = key_of(f.x, at.x);
      k[1] = key_of(f.y, at.y);
      k[2] = key_of(f.z, at.z);
      k[3] = key_of(f.w, at.w);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) k[e] = i + e < w_hi ? key_of(sc[i + e], pos[i + e]) : kNoKey;
    }
  };
  uint32_t held[TILES > 0 ? TILES : 1][4];
  // f(first slot of this lane, its 4 keys) for every tile of the warp, in order
  auto each_tile = [&](auto&& f) {
    if constexpr (TILES > 0) {
#pragma unroll
      for (int t = 0; t < TILES; ++t)
        if (w_lo + t * kTile < w_hi) f(w_lo + t * kTile + 4 * lane, held[t]);
    } else {
      for (int i0 = w_lo; i0 < w_hi; i0 += kTile) {
        uint32_t k[4];
        read4(i0 + 4 * lane, k);
        f(i0 + 4 * lane, k);
      }
    }
  };
  if constexpr (TILES > 0) {
#pragma unroll
    for (int t = 0; t < TILES; ++t)
      if (w_lo + t * kTile < w_hi) read4(w_lo + t * kTile + 4 * lane, held[t]);
  }

  // ---- the threshold: keys whose masked bits are above thr are kept, of those equal to it the
  // first `need`
  uint32_t thr = 0u, mask = 0u, need = uint32_t(p.budget);
  uint32_t rank_gt = 0u, rank_eq = 0u;       // warp r: CTA r's keys above and at thr
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t dmask = pass == 2 ? 1023u : 2047u;
    uint32_t* hist = s_hist[pass & 1];
    if (pass == 2) {
      // its readers of pass 0 have passed the barrier of pass 1
      *reinterpret_cast<uint4*>(hist + 4 * tid) = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
    }
    if (pass == 0) {
      // every key counts, without a branch
      each_tile([&](int, const uint32_t (&k)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          atomicAdd(hist + (k[e] == kNoKey ? uint32_t(kBins) : k[e] >> 21), 1u);
      });
    } else {
      each_tile([&](int, const uint32_t (&k)[4]) {
        bool in[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) in[e] = (k[e] & mask) == thr && k[e] != kNoKey;
        if (!__any_sync(kFullMask, in[0] || in[1] || in[2] || in[3])) return;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (in[e]) atomicAdd(hist + ((k[e] >> shift) & dmask), 1u);
      });
    }
    __syncthreads();
    // bins from the top: thread t owns the 4 bins from kBins - 4 - 4 t on
    uint4 c = *reinterpret_cast<const uint4*>(hist + kBins - 4 - 4 * tid);
    uint32_t sum = c.x + c.y + c.z + c.w, before = 0u, group_sum = 0u;
    int bin0 = kBins - 4 - 4 * tid, group = 0;
    if (C == 1) {
      sum = warp_inclusive(sum, lane);
      if (lane == 31) s_group[0][warp] = sum;
      __syncthreads();
      sum += sum_below(s_group[0], warp, lane);
    } else {
      // the CTAs' counts are joined in two steps, warp r fetching CTA r's: the groups of 128
      // bins, then the bins of the group where the count from the top reaches `need`
      sum = __reduce_add_sync(kFullMask, sum);
      if (lane == 0) s_group[pass & 1][warp] = sum;
      cluster.sync();
      if (warp < C && lane < kGroups) {
        group_sum = cluster.map_shared_rank(s_group[pass & 1], warp)[lane];
        s_groups[warp][lane] = group_sum;
      }
      __syncthreads();
      sum = 0u;
      if (lane < kGroups)
        for (int r = 0; r < C; ++r) sum += s_groups[r][lane];
      const uint32_t inc = warp_inclusive(sum, lane);
      group = __ffs(__ballot_sync(kFullMask, inc >= need)) - 1;   // the row has more keys
      before = __shfl_sync(kFullMask, inc - sum, group);
      bin0 = kBins - 128 * group - 4 - 4 * lane;
      if (warp < C) {
        c = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(hist, warp) + bin0);
        s_bins[warp][lane] = c;
      }
      __syncthreads();
    }
    if (C == 1 || warp == 0) {
      uint4 all = c;
      if (C > 1) {
        for (int r = 1; r < C; ++r) {
          const uint4 v = s_bins[r][lane];
          all.x += v.x; all.y += v.y; all.z += v.z; all.w += v.w;
        }
        sum = before + warp_inclusive(all.x + all.y + all.z + all.w, lane);
      }
      uint32_t above = sum - (all.x + all.y + all.z + all.w);
      if (above < need && sum >= need) {     // one thread
        const uint32_t bin[4] = {all.w, all.z, all.y, all.x};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (above < need && above + bin[e] >= need) {
            s_digit = uint32_t(bin0 + 3 - e);
            s_left = need - above;
            s_bin = bin[e];
          }
          above += bin[e];
        }
      }
    }
    __syncthreads();
    const uint32_t digit = s_digit;
    if (C > 1 && warp < C) {                 // CTA `warp`'s keys above and at the digit
      uint32_t up = lane < group ? group_sum : 0u, at = 0u;
      const uint32_t bin[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        up += uint32_t(bin0 + e) > digit ? bin[e] : 0u;
        at += uint32_t(bin0 + e) == digit ? bin[e] : 0u;
      }
      rank_gt += __reduce_add_sync(kFullMask, up);
      rank_eq = __reduce_add_sync(kFullMask, at);
    }
    thr |= digit << shift;
    mask |= dmask << shift;
    need = s_left;
    // the same in every CTA of the cluster: the whole bin is kept, or it holds one key only
    if (s_bin == need || (pass == 0 && (digit == kZeroBin || digit == kProtectedBin))) break;
  }
  // where the whole bin is kept, its keys count as above: no ties to rank (a bin at 0 holds NaN
  // scores and shares the value with the slots past the end)
  if (s_bin == need && thr != 0u) {
    thr -= 1u;
    need = 0u;
    rank_gt += rank_eq;
  }
  const bool ties = need > 0u;
  if (C > 1) {
    cluster.barrier_arrive();                // waited for at the end: no CTA ends while read
    if (warp < C && lane == 0) {
      s_rank_gt[warp] = rank_gt;
      s_rank_eq[warp] = rank_eq;
    }
  }

  // ---- keys above and at the threshold before each warp's slots
  uint32_t gt = 0u, eq = 0u;
  each_tile([&](int, const uint32_t (&k)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) gt += (k[e] & mask) > thr ? 1u : 0u;
    if (ties) {
#pragma unroll
      for (int e = 0; e < 4; ++e) eq += (k[e] & mask) == thr && k[e] != kNoKey ? 1u : 0u;
    }
  });
  gt = __reduce_add_sync(kFullMask, gt);
  eq = __reduce_add_sync(kFullMask, eq);
  if (lane == 0) {
    s_gt[warp] = gt;
    s_eq[warp] = eq;
  }
  __syncthreads();
  uint32_t gt_before = sum_below(s_gt, warp, lane);
  uint32_t eq_before = sum_below(s_eq, warp, lane);
  if (C > 1) {
    gt_before += sum_below(s_rank_gt, rank, lane);
    eq_before += sum_below(s_rank_eq, rank, lane);
  }

  // ---- the moves: the i-th hole from the front takes the i-th mover from the back
  const unsigned lower = (1u << lane) - 1u;
  const int last = p.budget - 1;
  each_tile([&](int i, const uint32_t (&k)[4]) {
    const int i0 = i - 4 * lane;
    bool kept[4], is_eq[4];
    unsigned above[4], at_thr[4];
    uint32_t gts = 0u, eqs = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      kept[e] = (k[e] & mask) > thr;
      above[e] = __ballot_sync(kFullMask, kept[e]);
      gts += __popc(above[e]);
    }
    if (ties) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        is_eq[e] = (k[e] & mask) == thr && k[e] != kNoKey;
        at_thr[e] = __ballot_sync(kFullMask, is_eq[e]);
        eqs += __popc(at_thr[e]);
      }
    }
    const uint32_t kept_eq = min(eq_before, need);
    const uint32_t here = gts + min(eq_before + eqs, need) - kept_eq;
    int g = int(gt_before + kept_eq);        // kept slots before this lane's, from the tile's on
    uint32_t q = eq_before;
    gt_before += gts;
    eq_before += eqs;
    // all movers and none kept, or all below the budget and none evicted: nothing to write
    if (i0 > last ? here == 0u : i0 + kTile <= last && here == uint32_t(kTile)) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) g += __popc(above[e] & lower);
    if (eqs) {
      const uint32_t q0 = q;
#pragma unroll
      for (int e = 0; e < 4; ++e) q += __popc(at_thr[e] & lower);
      g += int(min(q, need)) - int(min(q0, need));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        kept[e] = kept[e] || (is_eq[e] && q < need);
        q += is_eq[e] ? 1u : 0u;
      }
    }
    if (i0 > last) {                         // movers
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (kept[e]) src[last - g] = i + e;
        g += kept[e] ? 1 : 0;
      }
    } else if (i0 + kTile <= last) {         // holes (k is a slot's: the budget is below n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!kept[e]) dst[i + e - g] = i + e;
        g += kept[e] ? 1 : 0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = i + e;
        if (at <= last && !kept[e]) dst[at - g] = at;
        if (at > last && kept[e]) src[last - g] = at;
        if (at == last) p.counts[row] = p.budget - g - (kept[e] ? 1 : 0);
        g += kept[e] ? 1 : 0;
      }
    }
  });
  if (C > 1) cluster.barrier_wait();
}

// ------------------------------------------------------------------------------ compaction
//
// A warp takes up to 32 moves: each lane looks up one move's pages, so the chain of list, table
// and rows is paid once for all of them. Then kInFlight 16-byte loads a lane are issued before
// the first store; rows of at most 16 or 8 chunks share a warp's load. Bound by memory with rows of
// 256 bytes at random places: 229 MB (B=8, 16-32k slots to 4096, 8 heads of 128) in 43 us = 5.3
// TB/s of the 6.5 that a copy of one piece reaches; 4 rows a warp with a lookup each took 82 us,
// 4 / 16 loads in flight 46.7 / 45.5, 32 moves a warp 43.7, streaming cache hints 44.3. 16 moves
// a head (B=32) take 3.6 us, five dependent memory latencies and the launch.

constexpr int kMoveThreads = 256;
constexpr int kMoveWarps = kMoveThreads / 32;
constexpr int kInFlight = 8;
constexpr int kManyMoves = 16;   // moves of a warp when there are many

struct CacheView {
  uint8_t* base;
  int64_t sb, st, sh;       // bytes
  int row_bytes;
};

struct CompactParams {
  CacheView k, v;
  int64_t num_blocks;
  const int32_t* block_table;
  int64_t bt_sb;
  int max_blocks, block_size, bs_shift;
  const int32_t *src, *dst, *counts;
  int moves, kv_heads;
  float* scores;            // nullable
  int64_t sc_sb, sc_sh;
  int32_t* positions;       // nullable
  int64_t pos_sb, pos_sh;
  int slots;                // slots that a row of scores / positions has
  int lanes;                // lanes that copy a row: 8, 16 or 32
  int per_warp;             // moves of a warp, at most 32
  unsigned* status;         // nullable
};

__global__ void __launch_bounds__(kMoveThreads)
compact_kernel(const CompactParams p) {
  __shared__ int4 s_move[kMoveWarps][32];    // page and slot in it, from and to
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, b = blockIdx.z;
  const int i0 = (int(blockIdx.x) * kMoveWarps + warp) * p.per_warp;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = int64_t(b) * p.kv_heads + h;
  const int count = min(min(p.counts[row], p.moves) - i0, p.per_warp);
  if (count <= 0) return;
  const int64_t cap = min(int64_t(p.max_blocks) << p.bs_shift, int64_t(p.slots));
  const int32_t* bt = p.block_table + int64_t(b) * p.bt_sb;
  const int bmask = p.block_size - 1;
  if (lane < count) {
    const int from = p.src[row * p.moves + i0 + lane], to = p.dst[row * p.moves + i0 + lane];
    bool ok = from >= 0 && to >= 0;
    if (ok && (from >= cap || to >= cap)) {
      flag_device_error(p.status, BPT_DEV_SEQ_TOO_LONG);
      ok = false;
    }
    int pf = -1, pt = -1;
    if (ok) {
      pf = bt[from >> p.bs_shift];
      pt = bt[to >> p.bs_shift];
      if (pf < 0 || pf >= p.num_blocks || pt < 0 || pt >= p.num_blocks) {
        flag_device_error(p.status, BPT_DEV_BAD_BLOCK_ID);
        ok = false;
      }
    }
    s_move[warp][lane] = make_int4(ok ? pf : -1, from & bmask, pt, to & bmask);
    if (ok && p.scores) {
      float* s = p.scores + int64_t(b) * p.sc_sb + int64_t(h) * p.sc_sh;
      s[to] = s[from];
    }
    if (ok && p.positions) {
      int32_t* s = p.positions + int64_t(b) * p.pos_sb + int64_t(h) * p.pos_sh;
      s[to] = s[from];
    }
  }
  __syncwarp();
  const int sub = lane / p.lanes, step = 32 / p.lanes;   // rows that share a load
  const int kc = p.k.row_bytes >> 4, total = kc + (p.v.row_bytes >> 4);
  for (int m0 = sub; m0 < count; m0 += kInFlight * step)
    for (int c = lane % p.lanes; c < total; c += p.lanes) {
      const bool is_k = c < kc;
      const int64_t sb = is_k ? p.k.sb : p.v.sb, st = is_k ? p.k.st : p.v.st;
      uint8_t* col = (is_k ? p.k.base + int64_t(h) * p.k.sh : p.v.base + int64_t(h) * p.v.sh) +
                     16 * (is_k ? c : c - kc);
      uint4 d[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int m = m0 + u * step;
        if (m >= count) continue;
        const int4 v = s_move[warp][m];
        if (v.x >= 0) d[u] = *reinterpret_cast<const uint4*>(col + v.x * sb + v.y * st);
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int m = m0 + u * step;
        if (m >= count) continue;
        const int4 v = s_move[warp][m];
        if (v.x >= 0) *reinterpret_cast<uint4*>(col + v.z * sb + v.w * st) = d[u];
      }
    }
}

// ---------------------------------------------------------------------------------- append
//
// A token's K rows and V rows are copied 16 bytes a thread, U tokens of the same column at a
// time, the new rows asked for before the page table; where an address or stride is not a
// multiple of 16 bytes, 2 bytes a thread. Bound by memory: 101 MB (B=8, 1-2k tokens of 8 heads
// of 128) in 18.3 us = 5.5 TB/s; U = 4 / 8 / 16 took 18.7 / 19.7 / 25.2. One token of each of 64
// sequences takes 1.9 us, the launch and two memory latencies.

constexpr int kAppendThreads = 256;
constexpr int kPromptTokens = 2;   // U of an append of several tokens

struct AppendParams {
  CacheView k, v;           // paged: block, token, head
  CacheView kn, vn;         // new rows: sb = batch, st = token, sh = head
  int k_heads, v_heads;
  int64_t num_blocks;
  const int32_t* block_table;
  int64_t bt_sb;
  int max_blocks, block_size, bs_shift;
  const int32_t *new_lens, *seq_lens, *next_pos;
  int max_new;
  float* scores;            // nullable
  int64_t sc_sb, sc_sh;
  int32_t* positions;       // nullable
  int64_t pos_sb, pos_sh;
  unsigned* status;         // nullable
};

template <typename Word, int U>
__global__ void __launch_bounds__(kAppendThreads)
append_kernel(const AppendParams p) {
  constexpr int W = int(sizeof(Word));
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z;
  const int new_len = p.new_lens[b], start = p.seq_lens[b];
  const int m = min(max(new_len, 0), p.max_new), t0 = int(blockIdx.x) * U;
  // one thread a sequence, and before the CTAs without tokens leave
  if (new_len != m && (blockIdx.x | blockIdx.y | threadIdx.x) == 0)
    flag_device_error(p.status, BPT_DEV_BAD_NEW_LEN);
  if (t0 >= m) return;
  const int kw = p.k.row_bytes / W, vw = p.v.row_bytes / W;
  const int k_items = p.k_heads * kw, items = k_items + p.v_heads * vw;
  const int c = int(blockIdx.y) * kAppendThreads + int(threadIdx.x);
  const bool is_k = c < k_items;
  const int e = is_k ? c : c - k_items, w = is_k ? kw : vw;
  const int head = e / w, col = (e % w) * W;
  // the new rows do not wait for the table
  Word x[U];
  if (c < items) {
    const CacheView& from = is_k ? p.kn : p.vn;
    const uint8_t* f = from.base + int64_t(b) * from.sb + int64_t(t0) * from.st +
                       int64_t(head) * from.sh + col;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t0 + u < m) x[u] = *reinterpret_cast<const Word*>(f + int64_t(u) * from.st);
  }
  const int64_t cap = int64_t(p.max_blocks) << p.bs_shift;
  const int32_t* bt = p.block_table + int64_t(b) * p.bt_sb;
  int page[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t slot = int64_t(start) + t0 + u;
    page[u] = -1;
    if (t0 + u >= m) continue;
    if (slot < 0 || slot >= cap) {
      if (c == 0) flag_device_error(p.status, slot < 0 ? BPT_DEV_NEG_SEQ_LEN
                                                       : BPT_DEV_SEQ_TOO_LONG);
      continue;
    }
    page[u] = bt[slot >> p.bs_shift];
    if (page[u] < 0 || page[u] >= p.num_blocks) {
      if (c == 0) flag_device_error(p.status, BPT_DEV_BAD_BLOCK_ID);
      page[u] = -1;
    }
  }
  const int bmask = p.block_size - 1;
  if (c < items) {
    const CacheView& to = is_k ? p.k : p.v;
    uint8_t* d = to.base + int64_t(head) * to.sh + col;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (page[u] >= 0)
        *reinterpret_cast<Word*>(d + page[u] * to.sb + ((start + t0 + u) & bmask) * to.st) = x[u];
  }
  // the tokens' state: head h is thread h's (there are at least as many columns as heads)
  if (c >= p.v_heads) return;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (page[u] < 0) continue;
    const int64_t slot = int64_t(start) + t0 + u;
    if (p.scores) p.scores[int64_t(b) * p.sc_sb + int64_t(c) * p.sc_sh + slot] = 0.f;
    if (p.positions)
      p.positions[int64_t(b) * p.pos_sb + int64_t(c) * p.pos_sh + slot] =
          p.next_pos[b] + t0 + u;
  }
}

constexpr int kMaxGridYZ = 65535;
// Slots and moves are ints, and so are the ends of the last slice, tile or warp's moves, which pass
// them by less than this.
constexpr int kIndexRoom = 16384;
static_assert(kIndexRoom > 2 * kMaxCluster * kTile + 2 * kSelWarps * kTile &&
                  kIndexRoom > 32 * kMoveWarps,
              "slices and warps are rounded up to whole tiles");

int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

bool bad_cache(const bpt_paged_cache& c) {
  return c.k_heads <= 0 || c.v_heads <= 0 || c.k_dim <= 0 || c.v_dim <= 0 || c.num_blocks < 0 ||
         c.block_size <= 0 || !c.k || !c.v;
}

bool bad_pages(const bpt_paged_cache& c) {
  return c.block_size > 256 || (c.block_size & (c.block_size - 1));
}

CacheView view_of(void* base, const int64_t* stride, int dim) {
  CacheView v;
  v.base = static_cast<uint8_t*>(base);
  v.sb = stride[0] * 2;
  v.st = stride[1] * 2;
  v.sh = stride[2] * 2;
  v.row_bytes = dim * 2;
  return v;
}

struct Range {
  uintptr_t lo, hi;         // addresses, hi past the end
  bool meets(const Range& o) const { return lo < o.hi && o.lo < hi; }
};

Range words(const void* p, int64_t n) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  return {a, a + uintptr_t(n) * 4};
}

// Whether r meets a row of state [batch, heads, slots]. Rows are looked at one by one only where r
// lies between the first and the last of them.
bool meets_rows(const Range& r, const void* p, int64_t sb, int64_t sh, int batch, int heads,
                int slots) {
  if (slots == 0) return false;
  const char* base = static_cast<const char*>(p);
  const int64_t b1 = 4 * sb * (batch - 1), h1 = 4 * sh * (heads - 1);
  const char* low = base + (b1 < 0 ? b1 : 0) + (h1 < 0 ? h1 : 0);
  const char* high = base + (b1 > 0 ? b1 : 0) + (h1 > 0 ? h1 : 0);
  if (!r.meets({reinterpret_cast<uintptr_t>(low), words(high, slots).hi})) return false;
  for (int b = 0; b < batch; ++b)
    for (int h = 0; h < heads; ++h)
      if (r.meets(words(base + 4 * (b * sb + h * sh), slots))) return true;
  return false;
}

bool vec16(const CacheView& v) {
  return (reinterpret_cast<uintptr_t>(v.base) | uintptr_t(v.sb) | uintptr_t(v.st) |
          uintptr_t(v.sh) | uintptr_t(v.row_bytes)) % 16 == 0;
}

// CTAs per row: enough to put two on every SM, but at least kMinSlots slots a CTA, and more where
// a slice would not stay in registers.
int cluster_size(int64_t rows, int slots, int sms) {
  constexpr int kMinSlots = 2048;
  int c = 1;
  while (c < kMaxCluster &&
         ((rows * c <= sms && slots >= 2 * c * kMinSlots) ||
          slots > int64_t(c) * kMaxTiles * kTile * kSelWarps))
    c *= 2;
  return c;
}

}  // namespace
}  // namespace bpt

using namespace bpt;

extern "C" int bpt_evict_moves(int budget, int slots) {
  const int m = budget < slots - budget ? budget : slots - budget;
  return m < 1 ? 1 : m;
}

extern "C" int bpt_select_evictions(const float* scores, int64_t sc_sb, int64_t sc_sh,
                                    const int32_t* positions, int64_t pos_sb, int64_t pos_sh,
                                    const int32_t* seq_lens, const int32_t* next_pos, int batch,
                                    int kv_heads, int slots, int budget, int recent, int sinks,
                                    int32_t* src, int32_t* dst, int32_t* counts,
                                    int32_t* new_lens, void* stream) {
  if (batch < 0 || kv_heads <= 0 || slots < 0 || budget < 1 || recent < 0 || sinks < 0 ||
      int64_t(recent) + sinks > budget)
    return BPT_ERR_INVALID_ARGUMENT;
  if (batch == 0) return BPT_OK;
  if (!seq_lens || !next_pos || !src || !dst || !counts || !new_lens ||
      (slots > 0 && (!scores || !positions)))
    return BPT_ERR_INVALID_ARGUMENT;
  const int64_t rows = int64_t(batch) * kv_heads;
  // one CTA writes what others of the row have still to read: no result may lie on an input, nor
  // on another result
  const int64_t moves = bpt_evict_moves(budget, slots);
  const Range range[6] = {words(src, rows * moves), words(dst, rows * moves), words(counts, rows),
                          words(new_lens, batch), words(seq_lens, batch), words(next_pos, batch)};
  for (int i = 0; i < 4; ++i) {
    for (int j = i + 1; j < 6; ++j)
      if (range[i].meets(range[j])) return BPT_ERR_INVALID_ARGUMENT;
    if (meets_rows(range[i], scores, sc_sb, sc_sh, batch, kv_heads, slots) ||
        meets_rows(range[i], positions, pos_sb, pos_sh, batch, kv_heads, slots))
      return BPT_ERR_INVALID_ARGUMENT;
  }
  if (rows > INT32_MAX / kMaxCluster || slots > INT32_MAX - kIndexRoom)
    return BPT_ERR_UNSUPPORTED_SHAPE;
  const int C = cluster_size(rows, slots, device_sm_count());
  SelectParams p{};
  p.scores = scores;
  p.sc_sb = sc_sb;
  p.sc_sh = sc_sh;
  p.positions = positions;
  p.pos_sb = pos_sb;
  p.pos_sh = pos_sh;
  p.seq_lens = seq_lens;
  p.next_pos = next_pos;
  p.kv_heads = kv_heads;
  p.slots = slots;
  p.budget = budget;
  p.recent = recent;
  p.sinks = sinks;
  p.src = src;
  p.dst = dst;
  p.moves = int(moves);
  p.counts = counts;
  p.new_lens = new_lens;
  p.vec = ((reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(positions)) % 16 ==
           0) &&
          sc_sb % 4 == 0 && sc_sh % 4 == 0 && pos_sb % 4 == 0 && pos_sh % 4 == 0;
  // the kernel's own split of the longest row into slices and tiles
  const int per = cdiv(cdiv(slots, C), kTile) * kTile;
  const int tiles = cdiv(cdiv(per, kSelWarps), kTile);
  auto kern = tiles <= 1 ? select_kernel<1> : tiles <= 2 ? select_kernel<2>
            : tiles <= 4 ? select_kernel<4> : tiles <= 8 ? select_kernel<8>
            : tiles <= kMaxTiles ? select_kernel<kMaxTiles> : select_kernel<0>;
  if (C > 8 && cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) !=
                   cudaSuccess)
    return BPT_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * C));
  cfg.blockDim = dim3(kSelThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(C);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) return BPT_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? BPT_OK : BPT_ERR_LAUNCH;
}

extern "C" int bpt_compact_cache(const bpt_paged_cache* cache, const int32_t* block_table,
                                 int64_t bt_sb, int max_blocks, const int32_t* src,
                                 const int32_t* dst, const int32_t* counts, int moves, int batch,
                                 float* scores, int64_t sc_sb, int64_t sc_sh, int32_t* positions,
                                 int64_t pos_sb, int64_t pos_sh, int slots, unsigned* status,
                                 void* stream) {
  if (!cache || bad_cache(*cache) || batch < 0 || moves < 0 || max_blocks < 0 || slots < 0)
    return BPT_ERR_INVALID_ARGUMENT;
  if (cache->k_heads != cache->v_heads) return BPT_ERR_INVALID_ARGUMENT;
  if (bad_pages(*cache) || moves > INT32_MAX - kIndexRoom) return BPT_ERR_UNSUPPORTED_SHAPE;
  if (batch == 0 || moves == 0) return BPT_OK;
  if ((!block_table && max_blocks > 0) || !src || !dst || !counts) return BPT_ERR_INVALID_ARGUMENT;
  CompactParams p{};
  p.k = view_of(cache->k, cache->k_stride, cache->k_dim);
  p.v = view_of(cache->v, cache->v_stride, cache->v_dim);
  if (!vec16(p.k) || !vec16(p.v)) return BPT_ERR_ALIGNMENT;
  p.num_blocks = cache->num_blocks;
  p.block_table = block_table;
  p.bt_sb = bt_sb;
  p.max_blocks = max_blocks;
  p.block_size = cache->block_size;
  p.bs_shift = log2_of(cache->block_size);
  p.src = src;
  p.dst = dst;
  p.counts = counts;
  p.moves = moves;
  p.kv_heads = cache->k_heads;
  p.scores = scores;
  p.sc_sb = sc_sb;
  p.sc_sh = sc_sh;
  p.positions = positions;
  p.pos_sb = pos_sb;
  p.pos_sh = pos_sh;
  p.slots = scores || positions ? slots : INT32_MAX;
  p.status = status;
  if (p.kv_heads > kMaxGridYZ || batch > kMaxGridYZ) return BPT_ERR_UNSUPPORTED_SHAPE;
  const int chunks = (p.k.row_bytes + p.v.row_bytes) / 16;
  p.lanes = chunks > 16 ? 32 : chunks > 8 ? 16 : 8;
  // few moves: spread them over warps; many: pay the lookups once for two loads' worth
  const int at_once = kInFlight * (32 / p.lanes);
  p.per_warp = moves > 64 && at_once < kManyMoves ? kManyMoves : at_once;
  const int per_cta = kMoveWarps * p.per_warp;
  const dim3 grid(moves / per_cta + (moves % per_cta != 0), p.kv_heads, batch);
  if (launch_dependent(compact_kernel, grid, dim3(kMoveThreads), 0,
                       static_cast<cudaStream_t>(stream), p) != cudaSuccess)
    return BPT_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? BPT_OK : BPT_ERR_LAUNCH;
}

extern "C" int bpt_append_tokens(const bpt_paged_cache* cache, const void* k_new,
                                 const int64_t* kn_stride, const void* v_new,
                                 const int64_t* vn_stride, const int32_t* new_lens,
                                 const int32_t* seq_lens, const int32_t* block_table,
                                 int64_t bt_sb, int max_blocks, int batch, int max_new,
                                 float* scores, int64_t sc_sb, int64_t sc_sh,
                                 int32_t* positions, int64_t pos_sb, int64_t pos_sh,
                                 const int32_t* next_pos, unsigned* status, void* stream) {
  if (!cache || bad_cache(*cache) || batch < 0 || max_new < 0 || max_blocks < 0)
    return BPT_ERR_INVALID_ARGUMENT;
  if (bad_pages(*cache)) return BPT_ERR_UNSUPPORTED_SHAPE;
  // with no rows there is nothing to write, but lengths that ask for some are flagged
  if (batch == 0 || (max_new == 0 && !status)) return BPT_OK;
  if ((max_new > 0 && (!k_new || !v_new)) || !kn_stride || !vn_stride || !new_lens || !seq_lens ||
      (!block_table && max_blocks > 0) || (positions && !next_pos))
    return BPT_ERR_INVALID_ARGUMENT;
  AppendParams p{};
  p.k = view_of(cache->k, cache->k_stride, cache->k_dim);
  p.v = view_of(cache->v, cache->v_stride, cache->v_dim);
  p.kn = view_of(const_cast<void*>(k_new), kn_stride, cache->k_dim);
  p.vn = view_of(const_cast<void*>(v_new), vn_stride, cache->v_dim);
  p.k_heads = cache->k_heads;
  p.v_heads = cache->v_heads;
  p.num_blocks = cache->num_blocks;
  p.block_table = block_table;
  p.bt_sb = bt_sb;
  p.max_blocks = max_blocks;
  p.block_size = cache->block_size;
  p.bs_shift = log2_of(cache->block_size);
  p.new_lens = new_lens;
  p.seq_lens = seq_lens;
  p.next_pos = next_pos;
  p.max_new = max_new;
  p.scores = scores;
  p.sc_sb = sc_sb;
  p.sc_sh = sc_sh;
  p.positions = positions;
  p.pos_sb = pos_sb;
  p.pos_sh = pos_sh;
  p.status = status;
  const bool vec = vec16(p.k) && vec16(p.v) && vec16(p.kn) && vec16(p.vn);
  const int word = vec ? 16 : 2;
  const int64_t items = int64_t(p.k_heads) * (p.k.row_bytes / word) +
                        int64_t(p.v_heads) * (p.v.row_bytes / word);
  const int64_t blocks = (items + kAppendThreads - 1) / kAppendThreads;
  if (blocks > kMaxGridYZ || batch > kMaxGridYZ) return BPT_ERR_UNSUPPORTED_SHAPE;
  const int U = max_new == 1 ? 1 : kPromptTokens;
  const dim3 grid(max_new > 0 ? max_new / U + (max_new % U != 0) : 1, unsigned(blocks), batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kern = vec ? (U == 1 ? append_kernel<uint4, 1> : append_kernel<uint4, kPromptTokens>)
                  : (U == 1 ? append_kernel<uint16_t, 1>
                            : append_kernel<uint16_t, kPromptTokens>);
  const cudaError_t e = launch_dependent(kern, grid, dim3(kAppendThreads), 0, st, p);
  if (e != cudaSuccess) return BPT_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? BPT_OK : BPT_ERR_LAUNCH;
}
