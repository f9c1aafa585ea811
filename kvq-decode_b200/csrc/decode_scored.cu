// Decode attention that says what the cached tokens were worth: the scored decode and the
// differential decode over a paged fp16 / bf16 cache. No reference counterpart.
//
//   scored  x_gt = scale q_g.k_t, p_gt = exp(x_gt - max_t x) / sum_t exp(..)  (t < n)
//           out_g = sum_t p_gt v_t;  score_t <- decay * score_t + sum_g p_gt
//   diff    output head j has two q heads, two key heads and one value head of twice the width:
//           a_jt = p1_jt - lam_j p2_jt;  o_j = sum_t a_jt v_t;  with a norm weight
//           o_j <- o_j / sqrt(mean(o_j^2) + eps) * w;  out_j = out_scale * o_j
//           score_t <- decay * score_t + sum_j |a_jt|
//
// Two launches. The split kernel (mma_decode.cuh, OpState) is the fp16 decode's: one CTA per
// (sequence, kv head, split) reads K and V once for all the rows of the head. It also leaves
// every token's scaled logit in the workspace (4 bytes per row and token). A token's weight
// needs the sum over the whole sequence, known only when every split has ended, so the second
// kernel forms it: per row the splits' (max, sum) are joined, then 2^(x - M) / L of every token
// is added to its score, while other CTAs of the same launch join the splits' outputs. The
// logits cost 8 bytes a row and token (written and read, mostly in the 126 MB L2) where
// reading the keys again would cost 2 D a kv head and token.
#include <cuda_bf16.h>
#include <cudaTypedefs.h>
#include <float.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "decode_common.h"
#include "mma_decode.cuh"

namespace bpt {
namespace {

constexpr float kNegInf = -INFINITY;
constexpr int kFinishWarps = 8;
constexpr int kFinishThreads = kFinishWarps * 32;
constexpr int kScoreTokens = 4 * kFinishThreads;  // tokens of a round of a scoring CTA
constexpr int kMaxRows = 8;                       // q rows per kv head
static_assert(kMaxRows >= kFinishWarps, "shared rows double as one value a warp");
// A scoring CTA takes a further round of tokens for every kScoreCtas CTAs an SM that one round each
// would need: at least kScoreCtas and less than twice as many an SM are launched (the rounding of a
// row's parts aside). 29 us for 59 MB of logits with a CTA per 1024 tokens (4096 CTAs: B=16, 24-32k
// tokens, 32 q heads), 20 us with 512 or 768; the whole call at B=8, 12-16k tokens 81.4 us with 512
// CTAs of two rounds (3), 82.4 with 1024 of one (4 and more).
constexpr int kScoreCtas = 3;
// The logits stay in L2 (evict-last stores). A buffer that would be written back while the next
// call streams its cache is dropped line by line once read: 306 -> 298 us at 59 MB, 627 -> 620
// at 114 MB (B=16). At 17 MB dropping costs more than it saves: 89 -> 92 us (B=1, 128k tokens), the
// call alone. Smaller buffers so outlive the call in L2 at raised priority, up to a quarter of it.
constexpr int64_t kDropBytes = 32 << 20;

// Split CTA shape: 2 warps of 16 tokens each, and as many stages and CTAs an SM as keep about
// 200 KB of cache on its way: 160 (registers allow no more), 192 and 192 KB at 64, 128 and 256
// channels. Measured at B=8 and 0.47 GB of cache: width 64 with 3 stages and 4 CTAs 94 us, 4 and 5
// 89.5, 4 and 6 96.5, 6 and 4 92.6; width 256 with 64-token chunks in 2 stages and 1 CTA 107 us,
// 32-token chunks in 2 stages and 3 CTAs (registers spill) 100, 3 and 2 84.
constexpr int kSplitWarps = 2;
constexpr int kChunk = 16 * kSplitWarps;
constexpr int stages(int width) { return width == 64 ? 4 : 3; }
constexpr int resident_ctas(int width) { return width >= 256 ? 2 : width >= 128 ? 4 : 5; }

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct FinishParams {
  const float* m;       // [B, R, S] maxima (log2), R = rows per sequence
  const float* l;       // [B, R, S] sums
  const float* o_part;  // [B, R, S, D] normalised partial outputs
  const float* logits;  // [B, R, pitch]
  int64_t pitch;
  int drop_lines;       // drop the logits from L2 once read, instead of writing them back
  const int32_t* seq_lens;
  int64_t cap;
  float* scores;
  int64_t sc_sb, sc_sh;
  float decay;
  int score_vec;        // score rows are 16-byte aligned
  const float* lam;
  int64_t lam_sb, lam_sh;
  const float* norm_w;  // nullable, [D]
  float norm_eps, out_scale;
  void* out;
  int64_t o_sb, o_sh;
  int kv_heads, group, splits;
  int n_merge;          // CTAs [0, n_merge) join outputs, the others score tokens
  int out_heads;
  int rounds, parts;    // of a scoring CTA, scoring CTAs of a (sequence, kv head)
};

// (M, 1 / L) of one row over its S splits; every lane gets it. L = 0 (no token) gives 0.
__device__ __forceinline__ void row_state(const float* m, const float* l, int S, int lane,
                                          float& M, float& inv) {
  float mx = kNegInf, sum = 0.f;
  for (int s = lane; s < S; s += 32) {
    const float ms = m[s], ls = l[s];
    const float mn = fmaxf(mx, ms);
    if (mn != kNegInf) {
      sum = sum * fast_exp2(mx - mn) + ls * fast_exp2(ms - mn);
      mx = mn;
    } else {
      sum += ls;   // 0, or NaN of a NaN logit
    }
  }
  M = mx;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kFullMask, M, o));
  if (M == kNegInf) M = 0.f;
  float L = sum * fast_exp2(mx - M);
  if (mx == kNegInf) L = sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(kFullMask, L, o);
  inv = L == 0.f ? 0.f : 1.f / L;
}

template <bool BF16>
__device__ __forceinline__ void store16(void* base, int64_t at, float x) {
  if constexpr (BF16)
    static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(base)[at] = __float2half_rn(x);
}

// One output row (b, j): sum over its maps and splits of sign * (share of the split) * o. The
// warps are shared out to the maps; the first U rows of a warp are asked for before the row's
// state, so that 64 splits (32 of 256 channels) cost one memory round trip. 16 warps with DIFF, 8 a
// map, left one CTA an SM for the scoring: 83.4 us against 81.4 (B=8, 16k tokens, 4 value heads of
// 256).
template <int D, bool BF16, bool DIFF>
__device__ __forceinline__ void join_output(const FinishParams& p, int id, float* s_o,
                                            float* s_red) {
  constexpr int MAPS = DIFF ? 2 : 1;
  constexpr int WARPS = kFinishWarps / MAPS;       // of one map
  constexpr int V4 = (D + 127) / 128;             // float4 columns of a lane
  constexpr int U = MAPS * (V4 == 1 ? 8 : 4);     // rows in flight
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int map = warp / WARPS, w0 = warp % WARPS;
  const int b = id / p.out_heads, j = id % p.out_heads;
  const int S = p.splits;
  const int64_t row = (int64_t(b) * p.out_heads + j) * MAPS + map;
  const float* m = p.m + row * S;
  const float* l = p.l + row * S;
  const float* o = p.o_part + row * S * D;
  float4 acc[V4];
#pragma unroll
  for (int v = 0; v < V4; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = 0.f, inv = 0.f;
  for (int s0 = w0; s0 < S; s0 += WARPS * U) {
    float ms[U], ls[U];
    float4 x[U][V4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + WARPS * u;
      const bool in = s < S;
      ms[u] = in ? m[s] : 0.f;
      ls[u] = in ? l[s] : 0.f;
#pragma unroll
      for (int v = 0; v < V4; ++v) {
        const int c = 4 * (32 * v + lane);
        x[u][v] = (in && c < D) ? *reinterpret_cast<const float4*>(o + int64_t(s) * D + c)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    if (s0 == w0) {
      row_state(m, l, S, lane, M, inv);
      if (DIFF && map == 1) inv *= -p.lam[int64_t(b) * p.lam_sb + int64_t(j) * p.lam_sh];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float f = ls[u] == 0.f ? 0.f : fast_exp2(ms[u] - M) * ls[u] * inv;
#pragma unroll
      for (int v = 0; v < V4; ++v) {
        acc[v].x = fmaf(f, x[u][v].x, acc[v].x);
        acc[v].y = fmaf(f, x[u][v].y, acc[v].y);
        acc[v].z = fmaf(f, x[u][v].z, acc[v].z);
        acc[v].w = fmaf(f, x[u][v].w, acc[v].w);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V4; ++v) {
    const int c = 4 * (32 * v + lane);
    if (c < D) *reinterpret_cast<float4*>(s_o + warp * D + c) = acc[v];
  }
  __syncthreads();
  float r = 0.f;
  if (tid < D) {
#pragma unroll
    for (int w = 0; w < kFinishWarps; ++w) r += s_o[w * D + tid];
  }
  float mul = p.out_scale;
  if (DIFF && p.norm_w) {                         // uniform over the CTA
    const float w = tid < D ? p.norm_w[tid] : 0.f;
    float sq = r * r;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(kFullMask, sq, o);
    if (lane == 0) s_red[warp] = sq;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) total += s_red[k];
    // a row of zeros (an empty sequence is one) stays zeros with norm_eps 0 too
    mul *= total == 0.f ? 0.f : rsqrtf(total / float(D) + p.norm_eps) * w;
  }
  if (tid < D)
    store16<BF16>(p.out, int64_t(b) * p.o_sb + int64_t(j) * p.o_sh + tid, DIFF ? r * mul : r);
}

// The tokens of a CTA, all of one (sequence, kv head): p.rounds times 4 a thread. The first round's
// logits and old scores are asked for while the splits' states are joined, and with up to 4
// rows the next round's while this one is worked on. With 8 rows the second buffer's registers
// cost more than it hides: 349 us against 340 without (B=16, 24-32k tokens, 8 rows).
template <int ROWS, bool DIFF>
__device__ __forceinline__ void score_tokens(const FinishParams& p, int id, float* s_m,
                                             float* s_inv, float* s_lam) {
  constexpr int STEP = kScoreTokens;
  constexpr bool AHEAD = ROWS <= 4;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = id % p.parts, bh = id / p.parts;
  const int b = bh / p.kv_heads, h = bh % p.kv_heads;
  const int n = int(min(int64_t(max(p.seq_lens[b], 0)), p.cap));
  const int64_t first = int64_t(part) * p.rounds * STEP;
  if (first >= n) return;                         // uniform over the CTA
  const int64_t end = min(int64_t(n), first + int64_t(p.rounds) * STEP);
  const int G = p.group;
  const int64_t row0 = int64_t(bh) * G;
  const float* logits = p.logits + row0 * p.pitch;
  float* sc = p.scores + int64_t(b) * p.sc_sb + int64_t(h) * p.sc_sh;
  const bool fades = p.decay != 0.f;
  auto load = [&](int64_t t, float4 (&x)[ROWS], float4& old) {
    if (t >= end) return;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < G) x[r] = *reinterpret_cast<const float4*>(logits + r * p.pitch + t);
    if (fades && p.score_vec && t + 4 <= n) old = *reinterpret_cast<const float4*>(sc + t);
  };
  int64_t t = first + 4 * tid;
  float4 x[ROWS], old = make_float4(0.f, 0.f, 0.f, 0.f);
  load(t, x, old);
  if (warp < G) {
    float M, inv;
    row_state(p.m + (row0 + warp) * p.splits, p.l + (row0 + warp) * p.splits, p.splits, lane, M,
              inv);
    if (lane == 0) {
      s_m[warp] = M;
      s_inv[warp] = inv;
      if (DIFF)
        s_lam[warp] = p.lam[int64_t(b) * p.lam_sb + int64_t((h * G + warp) >> 1) * p.lam_sh];
    }
  }
  __syncthreads();
  for (; t - 4 * lane < end; t += STEP) {         // uniform over the warp
    float4 y[ROWS], next = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (AHEAD) load(t + STEP, y, next);
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    float a[4];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < G) {
        const float M = s_m[r], inv = s_inv[r];
        const float e[4] = {fast_exp2(x[r].x - M) * inv, fast_exp2(x[r].y - M) * inv,
                            fast_exp2(x[r].z - M) * inv, fast_exp2(x[r].w - M) * inv};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!DIFF) w[i] += e[i];
          else if ((r & 1) == 0) a[i] = e[i];
          else w[i] += fabsf(a[i] - s_lam[r] * e[i]);
        }
      }
    if (t >= end) {
      // past the last token of this lane
    } else if (p.score_vec && t + 4 <= n) {
      // decay 0 never reads the old scores: its `old` is 0
      *reinterpret_cast<float4*>(sc + t) =
          make_float4(fmaf(p.decay, old.x, w[0]), fmaf(p.decay, old.y, w[1]),
                      fmaf(p.decay, old.z, w[2]), fmaf(p.decay, old.w, w[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i < n) sc[t + i] = fades ? fmaf(p.decay, sc[t + i], w[i]) : w[i];
    }
    if (p.drop_lines) {                           // every lane of the warp has read its part
      __syncwarp();
      if ((lane & 7) == 0 && t < end) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (r < G) discard_line(logits + r * p.pitch + t);
      }
    }
    if constexpr (AHEAD) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) x[r] = y[r];
      old = next;
    } else {
      load(t + STEP, x, old);
    }
  }
}

template <int D, int ROWS, bool BF16, bool DIFF>
__global__ void __launch_bounds__(kFinishThreads)
finish_scored_kernel(const FinishParams p) {
  __shared__ __align__(16) float s_o[kFinishWarps * D];
  __shared__ float s_a[kMaxRows], s_b[kMaxRows], s_c[kMaxRows];
  pdl_wait();
  // the next call's split kernel may start launching; it waits for this grid's end
  pdl_launch_dependents();
  if (int(blockIdx.x) < p.n_merge)
    join_output<D, BF16, DIFF>(p, blockIdx.x, s_o, s_a);
  else
    score_tokens<ROWS, DIFF>(p, int(blockIdx.x) - p.n_merge, s_a, s_b, s_c);
}

template <int D, bool BF16, bool DIFF>
int launch_both(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& p,
                const FinishParams& f, cudaStream_t st) {
  constexpr int R = resident_ctas(D), N = stages(D);
  using Op = mma::OpState<BF16, DIFF>;
  const bool wide = p.group > 4;
  const int rc = wide ? mma::launch<D, kSplitWarps, N, R, true, Op>(tk, tv, p, st)
                      : mma::launch<D, kSplitWarps, N, R, false, Op>(tk, tv, p, st);
  if (rc) return rc;
  const int64_t grid = int64_t(f.n_merge) +
                       (f.scores ? int64_t(p.batch) * p.kv_heads * f.parts : 0);
  auto finish = wide ? finish_scored_kernel<D, 8, BF16, DIFF>
                     : finish_scored_kernel<D, 4, BF16, DIFF>;
  return launch_dependent(finish, dim3(unsigned(grid)), dim3(kFinishThreads), 0, st, f) ==
                 cudaSuccess
             ? BPT_OK
             : BPT_ERR_LAUNCH;
}

template <int D, bool DIFF>
int launch_typed(bool bf16, const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& p,
                 const FinishParams& f, cudaStream_t st) {
  return bf16 ? launch_both<D, true, DIFF>(tk, tv, p, f, st)
              : launch_both<D, false, DIFF>(tk, tv, p, f, st);
}

int64_t logit_pitch(int64_t cap) { return (cap + 63) / 64 * 64; }   // whole chunks, 16 bytes

struct ScoredView {
  unsigned* status;
  float *m, *l, *o_part, *logits;
  size_t bytes;
};

// [status word, padded][maxima][sums][partial outputs][logits], each padded to 256 bytes
ScoredView scored_view(void* ws, int batch, int rows, int width, int splits, int64_t tokens) {
  char* base = static_cast<char*>(ws);
  const size_t n = size_t(batch) * rows * splits;
  const size_t state = align256(n * sizeof(float));
  const size_t part = align256(n * width * sizeof(float));
  ScoredView v;
  v.status = reinterpret_cast<unsigned*>(base);
  v.m = reinterpret_cast<float*>(base + 256);
  v.l = reinterpret_cast<float*>(base + 256 + state);
  v.o_part = reinterpret_cast<float*>(base + 256 + 2 * state);
  v.logits = reinterpret_cast<float*>(base + 256 + 2 * state + part);
  v.bytes = 256 + 2 * state + part +
            (tokens > 0 ? size_t(batch) * rows * logit_pitch(tokens) * sizeof(float) : 0);
  return v;
}

// The shared planner's count, but one chunk a split where that still is one wave (the planner
// keeps two): B=1, 8 kv heads of 128, 512 / 1024 / 2048 tokens 6.3 / 6.6 / 7.5 us against 7.1 / 7.5
// / 8.1 with two (5.9 / 6.3 / 7.2 now).
int state_splits(int width, int batch, int kv_heads, int block_size, int max_blocks,
                 int num_splits, int sm_count) {
  const int resident = resident_ctas(width);
  int s = num_splits;
  if (s <= 0) {
    if (sm_count <= 0) sm_count = device_sm_count();
    const int64_t chunks = (int64_t(max_blocks) * block_size + kChunk - 1) / kChunk;
    s = chunks * batch * kv_heads <= int64_t(sm_count) * resident
            ? int(chunks)
            : plan_splits(batch, kv_heads, block_size, max_blocks, sm_count, resident, kChunk);
  }
  return clamp_splits(s, block_size, max_blocks, kChunk);
}

bool misaligned(const void* x, int bytes) { return reinterpret_cast<uintptr_t>(x) % bytes; }

}  // namespace
}  // namespace bpt

using namespace bpt;

extern "C" int bpt_effective_splits_scored(int head_dim, int maps, int batch, int kv_heads,
                                           int block_size, int max_blocks, int num_splits,
                                           int sm_count) {
  return state_splits(maps * head_dim, batch, kv_heads, block_size, max_blocks, num_splits,
                      sm_count);
}

extern "C" size_t bpt_scored_workspace_bytes(int head_dim, int maps, int batch, int q_heads,
                                             int splits, int64_t tokens) {
  if (batch <= 0 || q_heads <= 0 || head_dim <= 0 || splits <= 0 || maps <= 0) return 256;
  return scored_view(nullptr, batch, q_heads, maps * head_dim, splits, tokens).bytes;
}

extern "C" int bpt_decode_scored(const bpt_scored_decode* a, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (!a) return BPT_ERR_INVALID_ARGUMENT;
  const int maps = a->maps;
  if ((maps != 1 && maps != 2) || (a->dtype != BPT_FP16 && a->dtype != BPT_BF16))
    return BPT_ERR_INVALID_ARGUMENT;
  if (a->batch < 0 || a->kv_heads <= 0 || a->q_heads <= 0 || a->q_heads % (maps * a->kv_heads) ||
      a->block_size <= 0 || a->max_blocks < 0 || a->num_blocks < 0 || a->head_dim <= 0)
    return BPT_ERR_INVALID_ARGUMENT;
  // log2(e) * scale and the products with decay and norm_eps have to be numbers
  if (!(a->scale <= FLT_MAX / 2) || (a->scores && !(fabsf(a->decay) <= FLT_MAX)) ||
      (maps == 2 && a->norm_weight && !(a->norm_eps >= 0.f && a->norm_eps <= FLT_MAX)))
    return BPT_ERR_INVALID_ARGUMENT;
  if (a->batch == 0) return BPT_OK;
  if (!a->q || !a->k_cache || !a->v_cache || (!a->block_table && a->max_blocks > 0) ||
      !a->seq_lens || !a->out || !workspace || (maps == 2 && !a->lam))
    return BPT_ERR_INVALID_ARGUMENT;
  const int D = a->head_dim, width = maps * D;
  const int group = a->q_heads / a->kv_heads;
  if (group > kMaxRows || a->batch > 65535 || a->kv_heads > 65535)   // grid dimensions
    return BPT_ERR_UNSUPPORTED_SHAPE;
  if (!(width == 64 || width == 128 || width == 256) || D < 64) return BPT_ERR_UNSUPPORTED_SHAPE;
  if (a->block_size < 16 || a->block_size > 256 || (a->block_size & (a->block_size - 1)))
    return BPT_ERR_UNSUPPORTED_SHAPE;
  // q fragments are read as 4-byte pairs; outputs are single elements; the tensor maps check
  // the caches
  if (misaligned(a->q, 4) || a->q_stride[0] % 2 || a->q_stride[1] % 2) return BPT_ERR_ALIGNMENT;
  const int64_t cap = int64_t(a->max_blocks) * a->block_size;
  // the ends of the last chunk's tokens are ints
  if (cap > INT32_MAX - kChunk) return BPT_ERR_UNSUPPORTED_SHAPE;
  const int S = state_splits(width, a->batch, a->kv_heads, a->block_size, a->max_blocks,
                             a->num_splits, a->sm_count);
  const int64_t tokens = a->scores ? cap : 0;
  const ScoredView ws = scored_view(workspace, a->batch, a->q_heads, width, S, tokens);
  if (workspace_bytes < ws.bytes) return BPT_ERR_WORKSPACE_TOO_SMALL;
  if (misaligned(workspace, 16)) return BPT_ERR_ALIGNMENT;

  DecodeParams p{};
  const int box_rows = a->block_size < kChunk ? a->block_size : kChunk;
  const CUtensorMapDataType type = a->dtype == BPT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tk, tv;
  int rc = encode_kv_map(&tk, a->k_cache, type, 2, D, maps * a->kv_heads, a->block_size,
                         a->num_blocks, a->k_stride[2], a->k_stride[1], a->k_stride[0], 64,
                         box_rows, &p.k_c1, 128);
  if (rc) return rc;
  rc = encode_kv_map(&tv, a->v_cache, type, 2, width, a->kv_heads, a->block_size, a->num_blocks,
                     a->v_stride[2], a->v_stride[1], a->v_stride[0], 64, box_rows, &p.v_c1, 128);
  if (rc) return rc;
  p.q = static_cast<const __half*>(a->q);   // 16-bit elements, read as pairs
  p.q_sb = a->q_stride[0];
  p.q_sh = a->q_stride[1];
  p.block_table = a->block_table;
  p.bt_sb = a->bt_stride;
  p.seq_lens = a->seq_lens;
  p.o_part = ws.o_part;
  p.lse = ws.m;
  p.part_l = ws.l;
  p.logits = a->scores ? ws.logits : nullptr;
  p.logit_pitch = logit_pitch(cap);
  p.status = ws.status;
  p.batch = a->batch;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.group = group;
  p.splits = S;
  p.final_out = 0;
  p.balance = balanced_splits(a->batch, a->kv_heads, S, resident_ctas(width)) ? 1 : 0;
  p.block_size = a->block_size;
  p.max_blocks = a->max_blocks;
  p.box_rows = box_rows;
  p.num_blocks = a->num_blocks;
  const float sc = a->scale > 0.f ? a->scale : 1.0f / sqrtf(float(D));
  p.scale_log2 = sc * 1.4426950408889634f;

  FinishParams f{};
  f.m = ws.m;
  f.l = ws.l;
  f.o_part = ws.o_part;
  f.logits = ws.logits;
  f.pitch = p.logit_pitch;
  f.drop_lines = a->scores && !misaligned(ws.logits, 128) &&
                 int64_t(a->batch) * a->q_heads * f.pitch * 4 >= kDropBytes;
  f.seq_lens = a->seq_lens;
  f.cap = cap;
  f.scores = a->scores;
  f.sc_sb = a->scores_stride[0];
  f.sc_sh = a->scores_stride[1];
  f.decay = a->decay;
  f.score_vec = !misaligned(a->scores, 16) && f.sc_sb % 4 == 0 && f.sc_sh % 4 == 0;
  f.lam = a->lam;
  f.lam_sb = a->lam_stride[0];
  f.lam_sh = a->lam_stride[1];
  f.norm_w = a->norm_weight;
  f.norm_eps = a->norm_eps;
  f.out_scale = a->out_scale;
  f.out = a->out;
  f.o_sb = a->out_stride[0];
  f.o_sh = a->out_stride[1];
  f.kv_heads = a->kv_heads;
  f.group = group;
  f.splits = S;
  f.out_heads = a->q_heads / maps;
  f.n_merge = a->batch * f.out_heads;
  // rounds: one below 2 * kScoreCtas CTAs an SM, then what keeps them below that (floor)
  const int64_t steps = (cap + kScoreTokens - 1) / kScoreTokens;
  const int64_t rows = int64_t(a->batch) * a->kv_heads;
  const int64_t most = int64_t(kScoreCtas) * device_sm_count();
  f.rounds = int(std::max<int64_t>(1, std::min<int64_t>(steps, steps * rows / most)));
  f.parts = int((steps + f.rounds - 1) / f.rounds);
  if (f.n_merge + rows * f.parts > INT32_MAX) return BPT_ERR_UNSUPPORTED_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = a->dtype == BPT_BF16;
  if (maps == 2)
    rc = D == 64 ? launch_typed<128, true>(bf16, tk, tv, p, f, st)
                 : launch_typed<256, true>(bf16, tk, tv, p, f, st);
  else if (D == 64)
    rc = launch_typed<64, false>(bf16, tk, tv, p, f, st);
  else if (D == 128)
    rc = launch_typed<128, false>(bf16, tk, tv, p, f, st);
  else
    rc = launch_typed<256, false>(bf16, tk, tv, p, f, st);
  if (rc) return rc;
  return cudaGetLastError() == cudaSuccess ? BPT_OK : BPT_ERR_LAUNCH;
}
