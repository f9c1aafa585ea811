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
// to unsigned keys of the same order: three passes over 11 + 11 + 10 bits, each a histogram of
// the keys that share the digits found so far. One cluster of C CTAs takes one (sequence, kv
// head): each CTA reads its slice of the scores and positions once and keeps the keys in shared
// memory; histograms and prefix counts are exchanged through distributed shared memory. Ties
// at the threshold go to the lowest slots, so the result is unique and does not depend on the
// order in which the histogram's integer atomics arrive.

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kTile = 128;                   // slots of one vector load of a warp
constexpr int kMaxKeys = 48 * 1024;          // keys a CTA holds in shared memory (192 KB)
constexpr uint32_t kProtectedKey = 0xffffffffu;

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
  int key_cap;                               // keys that fit the launch's shared memory
  int vec;                                   // rows are 16-byte aligned
};

// Unsigned key of the same order as the score: NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t score_key(float f) {
  if (f != f) return 0u;
  const uint32_t u = __float_as_uint(f + 0.f);
  return u ^ ((u & 0x80000000u) ? 0xffffffffu : 0x80000000u);
}

__global__ void __launch_bounds__(kSelThreads)
select_kernel(const SelectParams p) {
  extern __shared__ __align__(16) uint32_t smem_sel[];
  uint32_t* s_keys = smem_sel + 2 * kBins;   // two histograms first
  __shared__ uint32_t s_scan[kSelWarps];
  __shared__ uint32_t s_digit, s_left;
  __shared__ uint32_t s_gt[kSelWarps], s_eq[kSelWarps];
  __shared__ uint32_t s_tot[2];              // this CTA's keys above and at the threshold

  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = int(blockIdx.x) / C;
  const int b = row / p.kv_heads, h = row % p.kv_heads;

  pdl_wait();
  pdl_launch_dependents();
  const int n = min(max(p.seq_lens[b], 0), p.slots);
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = min(n, p.budget);
  int32_t* src = p.src + int64_t(row) * p.moves;
  int32_t* dst = p.dst + int64_t(row) * p.moves;
  // unused places; the cluster barriers below order this before the moves of any CTA
  for (int i = rank * kSelThreads + tid; i < p.moves; i += C * kSelThreads) {
    src[i] = -1;
    dst[i] = -1;
  }
  if (n <= p.budget) {                       // the same n in every CTA of the cluster
    if (rank == 0 && tid == 0) p.counts[row] = 0;
    return;
  }

  // this CTA's slots [lo, hi) and this warp's [w_lo, w_hi) of them: whole tiles
  const int per = cdiv(cdiv(n, C), kTile) * kTile;
  const int lo = min(n, rank * per), hi = min(n, lo + per);
  const int w_per = cdiv(cdiv(per, kSelWarps), kTile) * kTile;
  const int w_lo = min(hi, lo + warp * w_per), w_hi = min(hi, w_lo + w_per);
  const float* sc = p.scores + int64_t(b) * p.sc_sb + int64_t(h) * p.sc_sh;
  const int32_t* pos = p.positions + int64_t(b) * p.pos_sb + int64_t(h) * p.pos_sh;
  // 64-bit: next_pos - recent may pass the int range
  const int64_t first_recent = int64_t(p.next_pos[b]) - p.recent;
  const int32_t sinks = p.sinks;
  auto key_of = [&](float f, int32_t at) {
    return (at < sinks || at >= first_recent) ? kProtectedKey : score_key(f);
  };
  const bool resident = per <= p.key_cap;    // else every pass reads the row again
  auto key_at = [&](int i) { return resident ? s_keys[i - lo] : key_of(sc[i], pos[i]); };

  for (int i = tid; i < 2 * kBins; i += kSelThreads) smem_sel[i] = 0u;
  if (resident) {
    if (p.vec) {
#pragma unroll 4
      for (int i = w_lo + 4 * lane; i < w_hi; i += kTile) {
        // rows are T long: the last vector may reach past n, within the row or not
        if (i + 4 <= w_hi) {
          const float4 f = *reinterpret_cast<const float4*>(sc + i);
          const int4 at = *reinterpret_cast<const int4*>(pos + i);
          *reinterpret_cast<uint4*>(s_keys + (i - lo)) =
              make_uint4(key_of(f.x, at.x), key_of(f.y, at.y), key_of(f.z, at.z),
                         key_of(f.w, at.w));
        } else {
          for (int e = i; e < w_hi; ++e) s_keys[e - lo] = key_of(sc[e], pos[e]);
        }
      }
    } else {
#pragma unroll 4
      for (int i = w_lo + lane; i < w_hi; i += 32) s_keys[i - lo] = key_of(sc[i], pos[i]);
    }
  }
  __syncthreads();

  // ---- the threshold key and how many keys equal to it are kept
  uint32_t prefix = 0u, mask = 0u, left = uint32_t(p.budget);
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t dmask = pass == 2 ? 1023u : 2047u;
    uint32_t* hist = smem_sel + (pass & 1) * kBins;
    if (pass == 2) {
      // its readers of pass 0 have passed the barrier of pass 1
      for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0u;
      __syncthreads();
    }
    for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t k = i < w_hi ? key_at(i) : 0u;
      const bool in = i < w_hi && (k & mask) == prefix;
      // the protected tokens come in long runs of one key: one atomic for the warp's
      const unsigned run = __ballot_sync(kFullMask, in && k == kProtectedKey);
      if (in && k != kProtectedKey) atomicAdd(hist + ((k >> shift) & dmask), 1u);
      if (run && lane == 0) atomicAdd(hist + dmask, uint32_t(__popc(run)));
    }
    cluster.sync();
    // bins from the top: thread t owns the 4 bins below kBins - 4 t
    const int bin0 = kBins - 4 - 4 * tid;
    uint4 sum = make_uint4(0u, 0u, 0u, 0u);
    for (int r = 0; r < C; ++r) {
      const uint4 v =
          *reinterpret_cast<const uint4*>(cluster.map_shared_rank(hist, r) + bin0);
      sum.x += v.x;
      sum.y += v.y;
      sum.z += v.z;
      sum.w += v.w;
    }
    const uint32_t mine = sum.x + sum.y + sum.z + sum.w;
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(kFullMask, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    uint32_t before = inc - mine;
    for (int w = 0; w < warp; ++w) before += s_scan[w];
    // the thread in whose bins the count reaches `left` (exactly one: the row has more keys)
    if (before < left && before + mine >= left) {
      const uint32_t c[4] = {sum.w, sum.z, sum.y, sum.x};
      uint32_t above = before;
      int e = 0;
      while (above + c[e] < left) above += c[e++];
      s_digit = uint32_t(bin0 + 3 - e);
      s_left = left - above;
    }
    __syncthreads();
    prefix |= s_digit << shift;
    mask |= dmask << shift;
    left = s_left;
  }
  const uint32_t thr = prefix, need = left;

  // ---- keys above and at the threshold before each warp's slots
  uint32_t gt = 0u, eq = 0u;
  for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t k = i < w_hi ? key_at(i) : 0u;
    gt += __popc(__ballot_sync(kFullMask, i < w_hi && k > thr));
    eq += __popc(__ballot_sync(kFullMask, i < w_hi && k == thr));
  }
  if (lane == 0) {
    s_gt[warp] = gt;
    s_eq[warp] = eq;
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t g = 0u, q = 0u;
    for (int w = 0; w < kSelWarps; ++w) {
      g += s_gt[w];
      q += s_eq[w];
    }
    s_tot[0] = g;
    s_tot[1] = q;
  }
  cluster.sync();
  uint32_t gt_before = 0u, eq_before = 0u;
  for (int r = 0; r < rank; ++r) {
    const uint32_t* t = cluster.map_shared_rank(s_tot, r);
    gt_before += t[0];
    eq_before += t[1];
  }
  cluster.sync();                            // no CTA ends while another reads its totals
  for (int w = 0; w < warp; ++w) {
    gt_before += s_gt[w];
    eq_before += s_eq[w];
  }

  // ---- the moves: the i-th hole from the front takes the i-th mover from the back
  const unsigned lower = (1u << lane) - 1u;
  for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
    const int i = i0 + lane;
    const bool in = i < w_hi;
    const uint32_t k = in ? key_at(i) : 0u;
    const unsigned g = __ballot_sync(kFullMask, in && k > thr);
    const unsigned q = __ballot_sync(kFullMask, in && k == thr);
    const uint32_t eq_at = eq_before + __popc(q & lower);
    const int kept_before = int(gt_before + __popc(g & lower) + min(eq_at, need));
    const bool kept = k > thr || (k == thr && eq_at < need);
    if (in) {
      if (i < p.budget && !kept) dst[i - kept_before] = i;
      if (i >= p.budget && kept) src[p.budget - 1 - kept_before] = i;
      if (i == p.budget - 1) p.counts[row] = p.budget - kept_before - (kept ? 1 : 0);
    }
    gt_before += __popc(g);
    eq_before += __popc(q);
  }
}

// ------------------------------------------------------------------------------ compaction
//
// One warp moves kRows rows: all their 16-byte loads are issued before the first store.

constexpr int kMoveThreads = 256;
constexpr int kRows = 4;

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
  unsigned* status;         // nullable
};

__global__ void __launch_bounds__(kMoveThreads)
compact_kernel(const CompactParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, b = blockIdx.z;
  const int i0 = (int(blockIdx.x) * (kMoveThreads / 32) + warp) * kRows;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = int64_t(b) * p.kv_heads + h;
  const int count = min(p.counts[row], p.moves);
  if (i0 >= count) return;
  const int64_t cap = min(int64_t(p.max_blocks) << p.bs_shift, int64_t(p.slots));
  const int32_t* bt = p.block_table + int64_t(b) * p.bt_sb;
  int from[kRows], to[kRows];
  int64_t pf[kRows], pt[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const bool in = i0 + u < count;
    from[u] = in ? p.src[row * p.moves + i0 + u] : -1;
    to[u] = in ? p.dst[row * p.moves + i0 + u] : -1;
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    bool ok = from[u] >= 0 && to[u] >= 0;
    if (ok && (from[u] >= cap || to[u] >= cap)) {
      if (lane == 0) flag_device_error(p.status, BPT_DEV_SEQ_TOO_LONG);
      ok = false;
    }
    pf[u] = ok ? bt[from[u] >> p.bs_shift] : -1;
    pt[u] = ok ? bt[to[u] >> p.bs_shift] : -1;
    if (ok && (pf[u] < 0 || pf[u] >= p.num_blocks || pt[u] < 0 || pt[u] >= p.num_blocks)) {
      if (lane == 0) flag_device_error(p.status, BPT_DEV_BAD_BLOCK_ID);
      ok = false;
    }
    if (!ok) pf[u] = -1;
  }
  const int bmask = p.block_size - 1;
  const int kc = p.k.row_bytes >> 4, total = kc + (p.v.row_bytes >> 4);
  for (int c = lane; c < total; c += 32) {
    const CacheView& x = c < kc ? p.k : p.v;
    uint8_t* col = x.base + int64_t(h) * x.sh + 16 * (c < kc ? c : c - kc);
    uint4 d[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u)
      if (pf[u] >= 0)
        d[u] = *reinterpret_cast<const uint4*>(col + pf[u] * x.sb + (from[u] & bmask) * x.st);
#pragma unroll
    for (int u = 0; u < kRows; ++u)
      if (pf[u] >= 0)
        *reinterpret_cast<uint4*>(col + pt[u] * x.sb + (to[u] & bmask) * x.st) = d[u];
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (lane != u || pf[u] < 0) continue;
    if (p.scores) {
      float* s = p.scores + int64_t(b) * p.sc_sb + int64_t(h) * p.sc_sh;
      s[to[u]] = s[from[u]];
    }
    if (p.positions) {
      int32_t* s = p.positions + int64_t(b) * p.pos_sb + int64_t(h) * p.pos_sh;
      s[to[u]] = s[from[u]];
    }
  }
}

// ---------------------------------------------------------------------------------- append
//
// A token's K rows and V rows are copied 16 bytes a thread, kUnroll tokens of the same column
// at a time; where an address or stride is not a multiple of 16 bytes, 2 bytes a thread.

constexpr int kAppendThreads = 256;
constexpr int kUnroll = 4;

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

template <typename Word>
__global__ void __launch_bounds__(kAppendThreads)
append_kernel(const AppendParams p) {
  constexpr int W = int(sizeof(Word));
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z;
  const int m = min(max(p.new_lens[b], 0), p.max_new);
  const int t0 = int(blockIdx.x) * kUnroll;
  if (t0 >= m) return;
  const int start = p.seq_lens[b];
  const int64_t cap = int64_t(p.max_blocks) << p.bs_shift;
  const int kw = p.k.row_bytes / W, vw = p.v.row_bytes / W;
  const int k_items = p.k_heads * kw, items = k_items + p.v_heads * vw;
  const int c = int(blockIdx.y) * kAppendThreads + int(threadIdx.x);
  const int32_t* bt = p.block_table + int64_t(b) * p.bt_sb;
  int64_t page[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
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
    const bool is_k = c < k_items;
    const CacheView& to = is_k ? p.k : p.v;
    const CacheView& from = is_k ? p.kn : p.vn;
    const int e = is_k ? c : c - k_items, w = is_k ? kw : vw;
    const int head = e / w, col = (e % w) * W;
    const uint8_t* f = from.base + int64_t(b) * from.sb + int64_t(head) * from.sh + col;
    uint8_t* d = to.base + int64_t(head) * to.sh + col;
    Word x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (page[u] >= 0) x[u] = *reinterpret_cast<const Word*>(f + int64_t(t0 + u) * from.st);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (page[u] >= 0)
        *reinterpret_cast<Word*>(d + page[u] * to.sb + ((start + t0 + u) & bmask) * to.st) = x[u];
    return;
  }
  const int h = c - items;                   // one thread a head for the token's state
  if (h >= p.v_heads) return;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (page[u] < 0) continue;
    const int64_t slot = int64_t(start) + t0 + u;
    if (p.scores) p.scores[int64_t(b) * p.sc_sb + int64_t(h) * p.sc_sh + slot] = 0.f;
    if (p.positions)
      p.positions[int64_t(b) * p.pos_sb + int64_t(h) * p.pos_sh + slot] =
          p.next_pos[b] + t0 + u;
  }
}

constexpr int kMaxGridYZ = 65535;

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

bool vec16(const CacheView& v) {
  return (reinterpret_cast<uintptr_t>(v.base) | uintptr_t(v.sb) | uintptr_t(v.st) |
          uintptr_t(v.sh) | uintptr_t(v.row_bytes)) % 16 == 0;
}

// CTAs per row: enough that the rows fill the SMs, but at least kMinSlots slots a CTA.
int cluster_size(int64_t rows, int slots, int sms) {
  constexpr int kMinSlots = 2048;
  int c = 1;
  while (c < 8 && ((rows * c * 2 <= sms && slots >= 2 * c * kMinSlots) ||
                   slots > int64_t(c) * kMaxKeys))
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
  if (!seq_lens || !next_pos || !src || !dst || !counts || !new_lens || seq_lens == new_lens ||
      (slots > 0 && (!scores || !positions)))
    return BPT_ERR_INVALID_ARGUMENT;
  const int64_t rows = int64_t(batch) * kv_heads;
  const int C = cluster_size(rows, slots, device_sm_count());
  if (rows * C > INT32_MAX) return BPT_ERR_UNSUPPORTED_SHAPE;
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
  p.moves = bpt_evict_moves(budget, slots);
  p.counts = counts;
  p.new_lens = new_lens;
  const int per = ((slots + C - 1) / C + kTile - 1) / kTile * kTile;
  p.key_cap = per < kMaxKeys ? per : kMaxKeys;
  p.vec = ((reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(positions)) % 16 ==
           0) &&
          sc_sb % 4 == 0 && sc_sh % 4 == 0 && pos_sb % 4 == 0 && pos_sh % 4 == 0;
  const size_t smem = size_t(2 * kBins + p.key_cap) * sizeof(uint32_t);
  if (cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int((2 * kBins + kMaxKeys) * sizeof(uint32_t))) != cudaSuccess)
    return BPT_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * C));
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = smem;
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
  if (cudaLaunchKernelEx(&cfg, select_kernel, p) != cudaSuccess) return BPT_ERR_LAUNCH;
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
  if (bad_pages(*cache)) return BPT_ERR_UNSUPPORTED_SHAPE;
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
  constexpr int kPerCta = kMoveThreads / 32 * kRows;
  const dim3 grid(moves / kPerCta + (moves % kPerCta != 0), p.kv_heads, batch);
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
  if (batch == 0 || max_new == 0) return BPT_OK;
  if (!k_new || !v_new || !kn_stride || !vn_stride || !new_lens || !seq_lens ||
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
                        int64_t(p.v_heads) * (p.v.row_bytes / word) + p.v_heads;
  const int64_t blocks = (items + kAppendThreads - 1) / kAppendThreads;
  if (blocks > kMaxGridYZ || batch > kMaxGridYZ) return BPT_ERR_UNSUPPORTED_SHAPE;
  const int groups = max_new / kUnroll + (max_new % kUnroll != 0);
  const dim3 grid(groups, unsigned(blocks), batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      vec ? launch_dependent(append_kernel<uint4>, grid, dim3(kAppendThreads), 0, st, p)
          : launch_dependent(append_kernel<uint16_t>, grid, dim3(kAppendThreads), 0, st, p);
  if (e != cudaSuccess) return BPT_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? BPT_OK : BPT_ERR_LAUNCH;
}
