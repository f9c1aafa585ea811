// Python binding of the scored decode and the eviction (bpt/evict.py, bpt/diff.py): argument
// checks, output allocation and the C-ABI call in one step.
//
// These calls run once per layer and token on a few microseconds of GPU work. Read from
// Python, the shapes, strides and pointers of their 6 to 12 tensors cost more than that:
// measured on the GPU host, 33 us a call through ctypes against 8 us here. The C ABI
// itself (include/bpt.h) stays free of torch; its functions reach this module by address, from
// the library that bpt._lib loaded.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <cfloat>
#include <cmath>
#include <optional>
#include <string>

#include "../../include/bpt.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Entry {
  decltype(&bpt_effective_splits_scored) effective_splits;
  decltype(&bpt_scored_workspace_bytes) workspace_bytes;
  decltype(&bpt_decode_scored) decode;
  decltype(&bpt_append_tokens) append;
  decltype(&bpt_evict_moves) evict_moves;
  decltype(&bpt_select_evictions) select;
  decltype(&bpt_compact_cache) compact;
} g_abi = {};
PyObject* g_argument_error = nullptr;   // bpt.BptArgumentError, kept for the process
PyObject* g_check = nullptr;            // bpt._lib.check: status -> exception

template <typename F>
void bind_to(F& fn, const py::dict& table, const char* name) {
  fn = reinterpret_cast<F>(table[name].cast<uintptr_t>());
}

[[noreturn]] void refuse(const std::string& why) {
  PyErr_SetString(g_argument_error ? g_argument_error : PyExc_RuntimeError, why.c_str());
  throw py::error_already_set();
}

void require_init() {
  if (__builtin_expect(!g_abi.compact, 0))
    refuse("bpt/_bind is used through bpt.evict and bpt.diff");
}

// The message is built only for a call that is refused.
#define REQUIRE(cond, ...)                       \
  do {                                           \
    if (__builtin_expect(!(cond), 0)) refuse(__VA_ARGS__); \
  } while (0)

void check(int status, const char* what) {
  if (__builtin_expect(status != BPT_OK, 0)) {
    PyObject* r = PyObject_CallFunction(g_check, "is", status, what);
    if (!r) throw py::error_already_set();
    Py_DECREF(r);
  }
}

std::string dims(std::initializer_list<int64_t> d) {
  std::string s = "[";
  for (int64_t x : d) s += (s.size() > 1 ? ", " : "") + std::to_string(x);
  return s + "]";
}

constexpr auto kI32 = at::ScalarType::Int;
constexpr auto kF32 = at::ScalarType::Float;

bool unit(const Tensor& t, int64_t dim) { return t.stride(dim) == 1 || t.size(dim) <= 1; }

template <typename T = void>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <typename T = void>
T* ptr(const OptTensor& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// Tensors that are written: no dimension may revisit the same memory.
void require_not_expanded(const Tensor& t, const char* name) {
  for (int64_t d = 0; d < t.dim(); ++d)
    REQUIRE(t.stride(d) != 0 || t.size(d) <= 1,
            std::string(name) + " is written and cannot be an expanded view");
}

struct Device {
  c10::Device dev;
  explicit Device(const Tensor& t) : dev(t.device()) {
    REQUIRE(dev.is_cuda(), "bpt runs on CUDA tensors only (no CPU fallback)");
  }
  void same(const Tensor& t, const char* name) const {
    REQUIRE(t.device() == dev, std::string(name) + " is on " + t.device().str() + ", not on " +
                                   dev.str());
  }
  void same(const OptTensor& t, const char* name) const {
    if (t) same(*t, name);
  }
};

struct Cache {
  int64_t num_blocks, block_size, k_heads, v_heads, k_dim, v_dim;
  bool bf16;
};

Cache check_cache(const Tensor& k, const Tensor& v) {
  REQUIRE(k.dim() == 4 && v.dim() == 4 && k.size(0) == v.size(0) && k.size(1) == v.size(1),
          "k_cache/v_cache must be [num_blocks, block_size, heads, D] of the same pages");
  const auto type = k.scalar_type();
  REQUIRE(type == v.scalar_type() &&
              (type == at::ScalarType::Half || type == at::ScalarType::BFloat16),
          "k_cache and v_cache must both be float16 or both bfloat16");
  REQUIRE(unit(k, 3) && unit(v, 3), "innermost (head_dim) stride must be 1");
  const int64_t bs = k.size(1);
  REQUIRE(bs >= 16 && (bs & (bs - 1)) == 0, "block_size must be a power of two >= 16");
  REQUIRE(k.size(2) > 0 && v.size(2) > 0 && k.size(3) > 0 && v.size(3) > 0,
          "k_cache/v_cache must have heads and channels");
  return {k.size(0), bs, k.size(2), v.size(2), k.size(3), v.size(3),
          type == at::ScalarType::BFloat16};
}

void check_table(const Tensor& bt, int64_t B) {
  REQUIRE(bt.dim() == 2 && bt.size(0) == B && bt.scalar_type() == kI32 && unit(bt, 1),
          "block_table must be int32 [B, max_blocks] with contiguous rows");
}

void check_lens(const Tensor& t, int64_t B, const char* name) {
  REQUIRE(t.dim() == 1 && t.size(0) == B && t.scalar_type() == kI32 && unit(t, 0),
          std::string(name) + " must be contiguous int32 [B]");
}

// A row of state per (sequence, kv head): [B, H, >= slots], unit inner stride.
void check_state(const Tensor& t, const char* name, at::ScalarType type, int64_t B, int64_t H,
                 int64_t slots, bool written) {
  REQUIRE(t.dim() == 3 && t.size(0) == B && t.size(1) == H && t.scalar_type() == type &&
              t.size(2) >= slots && unit(t, 2),
          std::string(name) + " must be " + (type == kF32 ? "float32" : "int32") + " [" +
              std::to_string(B) + ", " + std::to_string(H) + ", >= " + std::to_string(slots) +
              "] with a unit inner stride");
  if (written) require_not_expanded(t, name);
}

struct State {
  void* p = nullptr;
  int64_t sb = 0, sh = 0;
  State() = default;
  explicit State(const OptTensor& t) {
    if (t) {
      p = t->data_ptr();
      sb = t->stride(0);
      sh = t->stride(1);
    }
  }
};

bpt_paged_cache cache_c(const Tensor& k, const Tensor& v, const Cache& c) {
  bpt_paged_cache r;
  r.block_size = int(c.block_size);
  r.k_heads = int(c.k_heads);
  r.v_heads = int(c.v_heads);
  r.k_dim = int(c.k_dim);
  r.v_dim = int(c.v_dim);
  r.num_blocks = c.num_blocks;
  r.k = k.data_ptr();
  r.v = v.data_ptr();
  for (int i = 0; i < 3; ++i) {
    r.k_stride[i] = k.stride(i);
    r.v_stride[i] = v.stride(i);
  }
  return r;
}

// ------------------------------------------------------------------------------- entry points

int64_t scored_workspace_bytes(int maps, const Tensor& q, const Tensor& k_cache,
                               const Tensor& block_table, int num_splits, bool scored) {
  require_init();
  REQUIRE(q.dim() == 3 && k_cache.dim() == 4 && block_table.dim() == 2,
          "q must be [B, heads, D], k_cache [num_blocks, block_size, heads, D], block_table "
          "[B, max_blocks]");
  REQUIRE(maps == 1 || maps == 2, "maps must be 1 (scored) or 2 (differential)");
  REQUIRE(k_cache.size(2) > 0 && k_cache.size(2) % maps == 0 && q.size(1) > 0 && q.size(2) > 0,
          "k_cache must have maps heads for each kv head, q heads and channels");
  const int B = int(q.size(0)), Hq = int(q.size(1)), D = int(q.size(2));
  const int bs = int(k_cache.size(1)), mb = int(block_table.size(1));
  const c10::cuda::OptionalCUDAGuard guard(q.is_cuda() ? c10::optional<c10::Device>(q.device())
                                                       : c10::nullopt);
  const int S = g_abi.effective_splits(D, maps, B, int(k_cache.size(2)) / maps, bs, mb, num_splits,
                                       0);
  return int64_t(g_abi.workspace_bytes(D, maps, B, Hq, S, scored ? int64_t(mb) * bs : 0));
}

Tensor decode_scored(int maps, const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                     const Tensor& block_table, const Tensor& seq_lens,
                     std::optional<double> scale, std::optional<int> num_splits,
                     const OptTensor& scores, double decay, const OptTensor& out_arg,
                     const OptTensor& workspace_arg, const OptTensor& lam,
                     const OptTensor& norm_weight, double norm_eps, double out_scale) {
  require_init();
  REQUIRE(q.dim() == 3 && unit(q, 2), "q must be [B, heads, D] with a unit inner stride");
  const Cache c = check_cache(k_cache, v_cache);
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), H = c.v_heads;
  const int64_t width = maps * D;
  REQUIRE(q.scalar_type() == k_cache.scalar_type(), "q and the caches must have the same dtype");
  REQUIRE(c.k_heads == maps * H,
          "k_cache must have " + std::to_string(maps) + " heads for each head of v_cache");
  REQUIRE(c.k_dim == D && c.v_dim == width, "head_dim of q and the caches do not match");
  REQUIRE(Hq > 0 && Hq % (maps * H) == 0, "q heads must be a multiple of the key heads");
  check_table(block_table, B);
  check_lens(seq_lens, B, "seq_lens");
  const int64_t max_blocks = block_table.size(1), cap = max_blocks * c.block_size;
  REQUIRE(cap <= INT32_MAX && B <= 65535, "more than 2^31 slots or 65535 sequences");
  const int64_t out_heads = Hq / maps;
  if (scores) check_state(*scores, "scores", kF32, B, H, cap, true);
  // as the kernels take them: a scale that is 0 in fp32 would mean the default one
  REQUIRE(std::isfinite(float(decay)) && decay >= 0.0, "decay must be finite and not negative");
  REQUIRE(!scale || (float(*scale) > 0.f && float(*scale) <= FLT_MAX / 2),
          "scale must be positive and finite in fp32");
  if (maps == 2) {
    REQUIRE(lam && lam->scalar_type() == kF32 &&
                ((lam->dim() == 1 && lam->size(0) == out_heads) ||
                 (lam->dim() == 2 && lam->size(0) == B && lam->size(1) == out_heads)),
            "lam must be float32 " + dims({out_heads}) + " or " + dims({B, out_heads}));
    REQUIRE(!norm_weight || (norm_weight->dim() == 1 && norm_weight->size(0) == width &&
                             norm_weight->scalar_type() == kF32 && unit(*norm_weight, 0)),
            "norm_weight must be contiguous float32 " + dims({width}));
    REQUIRE(norm_eps >= 0.0 && std::isfinite(float(norm_eps)),
            "norm_eps must be finite and not negative");
  }
  const Device on(q);
  on.same(k_cache, "k_cache");
  on.same(v_cache, "v_cache");
  on.same(block_table, "block_table");
  on.same(seq_lens, "seq_lens");
  on.same(scores, "scores");
  on.same(lam, "lam");
  on.same(norm_weight, "norm_weight");
  on.same(out_arg, "out");
  on.same(workspace_arg, "workspace");
  if (out_arg) {
    REQUIRE(out_arg->dim() == 3 && out_arg->size(0) == B && out_arg->size(1) == out_heads &&
                out_arg->size(2) == width && out_arg->scalar_type() == q.scalar_type() &&
                unit(*out_arg, 2),
            "out must be of q's dtype, " + dims({B, out_heads, width}) +
                " with a unit inner stride");
    require_not_expanded(*out_arg, "out");
  }
  const c10::cuda::CUDAGuard guard(on.dev);
  const int ns = num_splits.value_or(0);
  const int S = g_abi.effective_splits(int(D), maps, int(B), int(H), int(c.block_size),
                                       int(max_blocks), ns, 0);
  const size_t need =
      g_abi.workspace_bytes(int(D), maps, int(B), int(Hq), S, scores ? cap : 0);
  Tensor out = out_arg ? *out_arg : at::empty({B, out_heads, width}, q.options());
  // without a workspace: memory of this stream's pool, given back (in stream order) on return
  void* ws = nullptr;
  size_t ws_bytes = need;
  c10::DataPtr own_ws;
  if (workspace_arg && workspace_arg->nbytes() >= need) {
    REQUIRE(workspace_arg->is_contiguous(), "workspace must be contiguous");
    ws = workspace_arg->data_ptr();
    ws_bytes = workspace_arg->nbytes();
  } else {
    own_ws = c10::cuda::CUDACachingAllocator::get()->allocate(need);
    ws = own_ws.get();
  }
  bpt_scored_decode a = {};
  a.dtype = c.bf16 ? BPT_BF16 : BPT_FP16;
  a.maps = maps;
  a.batch = int(B);
  a.q_heads = int(Hq);
  a.kv_heads = int(H);
  a.head_dim = int(D);
  a.block_size = int(c.block_size);
  a.max_blocks = int(max_blocks);
  a.num_splits = ns;
  a.scale = float(scale.value_or(0.0));
  a.decay = float(decay);
  a.norm_eps = float(norm_eps);
  a.out_scale = float(out_scale);
  a.num_blocks = c.num_blocks;
  a.q = q.data_ptr();
  a.q_stride[0] = q.stride(0);
  a.q_stride[1] = q.stride(1);
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  for (int i = 0; i < 3; ++i) {
    a.k_stride[i] = k_cache.stride(i);
    a.v_stride[i] = v_cache.stride(i);
  }
  a.block_table = ptr<int32_t>(block_table);
  a.bt_stride = block_table.stride(0);
  a.seq_lens = ptr<int32_t>(seq_lens);
  a.out = out.data_ptr();
  a.out_stride[0] = out.stride(0);
  a.out_stride[1] = out.stride(1);
  const State sc(scores);
  a.scores = static_cast<float*>(sc.p);
  a.scores_stride[0] = sc.sb;
  a.scores_stride[1] = sc.sh;
  if (lam) {
    a.lam = ptr<float>(*lam);
    a.lam_stride[0] = lam->dim() == 2 ? lam->stride(0) : 0;
    a.lam_stride[1] = lam->stride(-1);
  }
  a.norm_weight = ptr<float>(norm_weight);
  check(g_abi.decode(&a, ws, ws_bytes,
                     c10::cuda::getCurrentCUDAStream(on.dev.index()).stream()),
        "bpt_decode_scored");
  return out;
}

void append_tokens(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_new,
                   const Tensor& v_new, const Tensor& new_lens, const Tensor& seq_lens,
                   const Tensor& block_table, const OptTensor& scores, const OptTensor& positions,
                   const OptTensor& next_pos, const OptTensor& status) {
  require_init();
  const Cache c = check_cache(k_cache, v_cache);
  REQUIRE(k_new.dim() == 4 && v_new.dim() == 4 && k_new.size(0) == v_new.size(0) &&
              k_new.size(1) == v_new.size(1) && k_new.size(2) == c.k_heads &&
              v_new.size(2) == c.v_heads && k_new.size(3) == c.k_dim && v_new.size(3) == c.v_dim,
          "k_new/v_new must be [B, S, heads, D] with the heads and widths of their caches");
  REQUIRE(k_new.scalar_type() == k_cache.scalar_type() &&
              v_new.scalar_type() == k_cache.scalar_type(),
          "k_new/v_new must have the cache's dtype");
  REQUIRE(unit(k_new, 3) && unit(v_new, 3), "k_new/v_new need a unit inner stride");
  const int64_t B = k_new.size(0), S = k_new.size(1), H = c.v_heads;
  REQUIRE(S <= INT32_MAX && B <= 65535, "more than 2^31 tokens or 65535 sequences");
  check_lens(new_lens, B, "new_lens");
  check_lens(seq_lens, B, "seq_lens");
  check_table(block_table, B);
  const int64_t cap = block_table.size(1) * c.block_size;
  if (scores) check_state(*scores, "scores", kF32, B, H, cap, true);
  if (positions) {
    check_state(*positions, "positions", kI32, B, H, cap, true);
    REQUIRE(next_pos, "positions need next_pos");
  }
  if (next_pos) check_lens(*next_pos, B, "next_pos");
  require_not_expanded(k_cache, "k_cache");
  require_not_expanded(v_cache, "v_cache");
  const Device on(k_cache);
  on.same(v_cache, "v_cache");
  on.same(k_new, "k_new");
  on.same(v_new, "v_new");
  on.same(new_lens, "new_lens");
  on.same(seq_lens, "seq_lens");
  on.same(block_table, "block_table");
  on.same(scores, "scores");
  on.same(positions, "positions");
  on.same(next_pos, "next_pos");
  const c10::cuda::CUDAGuard guard(on.dev);
  const bpt_paged_cache cc = cache_c(k_cache, v_cache, c);
  const int64_t ks[3] = {k_new.stride(0), k_new.stride(1), k_new.stride(2)};
  const int64_t vs[3] = {v_new.stride(0), v_new.stride(1), v_new.stride(2)};
  const State sc(scores), pos(positions);
  check(g_abi.append(&cc, k_new.data_ptr(), ks, v_new.data_ptr(), vs, ptr<int32_t>(new_lens),
                     ptr<int32_t>(seq_lens), ptr<int32_t>(block_table), block_table.stride(0),
                     int(block_table.size(1)), int(B), int(S), static_cast<float*>(sc.p), sc.sb,
                     sc.sh, static_cast<int32_t*>(pos.p), pos.sb, pos.sh, ptr<int32_t>(next_pos),
                     ptr<unsigned>(status),
                     c10::cuda::getCurrentCUDAStream(on.dev.index()).stream()),
        "bpt_append_tokens");
}

// moves: a tuple (src, dst, counts, new_lens) to reuse, or None; returns such a tuple.
py::tuple select_evictions(const Tensor& scores, const Tensor& positions, const Tensor& seq_lens,
                           const Tensor& next_pos, int64_t budget, int64_t recent, int64_t sinks,
                           const std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>>& moves) {
  require_init();
  REQUIRE(scores.dim() == 3, "scores must be [B, Hkv, T]");
  const int64_t B = scores.size(0), H = scores.size(1), T = scores.size(2);
  check_state(scores, "scores", kF32, B, H, 0, false);
  check_state(positions, "positions", kI32, B, H, 0, false);
  REQUIRE(positions.size(2) == T, "scores and positions must have the same slots");
  check_lens(seq_lens, B, "seq_lens");
  check_lens(next_pos, B, "next_pos");
  REQUIRE(budget >= 1 && budget <= INT32_MAX && recent >= 0 && sinks >= 0 &&
              recent <= budget - (sinks < budget ? sinks : budget) && sinks <= budget,
          "budget must be an int32 of at least 1 and at least recent + sinks");
  REQUIRE(T <= INT32_MAX && H > 0, "scores must have kv heads and fewer than 2^31 slots");
  const Device on(scores);
  on.same(positions, "positions");
  on.same(seq_lens, "seq_lens");
  on.same(next_pos, "next_pos");
  const c10::cuda::CUDAGuard guard(on.dev);
  const int64_t M = g_abi.evict_moves(int(budget), int(T));
  Tensor src, dst, counts, new_lens;
  if (moves) {
    std::tie(src, dst, counts, new_lens) = *moves;
    const auto is = [&](const Tensor& t, std::initializer_list<int64_t> d, const char* name) {
      REQUIRE(t.sizes() == at::IntArrayRef(d) && t.scalar_type() == kI32 && t.is_contiguous(),
              std::string("moves.") + name + " must be contiguous int32 " + dims(d));
      on.same(t, name);
    };
    is(src, {B, H, M}, "src");
    is(dst, {B, H, M}, "dst");
    is(counts, {B, H}, "counts");
    is(new_lens, {B}, "new_lens");
    REQUIRE(B == 0 || (new_lens.data_ptr() != seq_lens.data_ptr() &&
                       new_lens.data_ptr() != next_pos.data_ptr()),
            "moves.new_lens cannot be seq_lens or next_pos itself");
  } else {
    // one allocation: src, dst, counts, new_lens
    const int64_t rows = B * H;
    const Tensor all = at::empty({2 * rows * M + rows + B}, seq_lens.options());
    src = all.as_strided({B, H, M}, {H * M, M, 1}, 0);
    dst = all.as_strided({B, H, M}, {H * M, M, 1}, rows * M);
    counts = all.as_strided({B, H}, {H, 1}, 2 * rows * M);
    new_lens = all.as_strided({B}, {1}, 2 * rows * M + rows);
  }
  check(g_abi.select(ptr<float>(scores), scores.stride(0), scores.stride(1),
                     ptr<int32_t>(positions), positions.stride(0), positions.stride(1),
                     ptr<int32_t>(seq_lens), ptr<int32_t>(next_pos), int(B), int(H), int(T),
                     int(budget), int(recent), int(sinks), ptr<int32_t>(src), ptr<int32_t>(dst),
                     ptr<int32_t>(counts), ptr<int32_t>(new_lens),
                     c10::cuda::getCurrentCUDAStream(on.dev.index()).stream()),
        "bpt_select_evictions");
  return py::make_tuple(src, dst, counts, new_lens);
}

void compact_cache(const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                   const Tensor& src, const Tensor& dst, const Tensor& counts,
                   const OptTensor& scores, const OptTensor& positions, const OptTensor& status) {
  require_init();
  const Cache c = check_cache(k_cache, v_cache);
  REQUIRE(c.k_heads == c.v_heads, "k_cache and v_cache must have the same heads");
  const int64_t H = c.v_heads;
  REQUIRE(src.dim() == 3 && src.size(1) == H && src.sizes() == dst.sizes() &&
              counts.dim() == 2 && counts.size(0) == src.size(0) && counts.size(1) == H,
          "moves must be src/dst [B, Hkv, M], counts [B, Hkv]");
  const int64_t B = src.size(0), M = src.size(2);
  REQUIRE(M <= INT32_MAX && B <= 65535, "more than 2^31 moves or 65535 sequences");
  for (const Tensor* t : {&src, &dst, &counts})
    REQUIRE(t->scalar_type() == kI32 && t->is_contiguous(), "moves must be contiguous int32");
  check_table(block_table, B);
  int64_t slots = block_table.size(1) * c.block_size;
  if (scores) {
    check_state(*scores, "scores", kF32, B, H, 0, true);
    slots = std::min(slots, scores->size(2));
  }
  if (positions) {
    check_state(*positions, "positions", kI32, B, H, 0, true);
    slots = std::min(slots, positions->size(2));
  }
  require_not_expanded(k_cache, "k_cache");
  require_not_expanded(v_cache, "v_cache");
  const Device on(k_cache);
  on.same(v_cache, "v_cache");
  on.same(block_table, "block_table");
  on.same(scores, "scores");
  on.same(positions, "positions");
  on.same(src, "moves.src");
  on.same(dst, "moves.dst");
  on.same(counts, "moves.counts");
  const c10::cuda::CUDAGuard guard(on.dev);
  const bpt_paged_cache cc = cache_c(k_cache, v_cache, c);
  const State sc(scores), pos(positions);
  check(g_abi.compact(&cc, ptr<int32_t>(block_table), block_table.stride(0),
                      int(block_table.size(1)), ptr<int32_t>(src), ptr<int32_t>(dst),
                      ptr<int32_t>(counts), int(M), int(B), static_cast<float*>(sc.p), sc.sb,
                      sc.sh, static_cast<int32_t*>(pos.p), pos.sb, pos.sh,
                      int(std::min<int64_t>(slots, INT32_MAX)), ptr<unsigned>(status),
                      c10::cuda::getCurrentCUDAStream(on.dev.index()).stream()),
        "bpt_compact_cache");
}

void init(const py::dict& abi, const py::object& argument_error, const py::object& check_fn) {
  bind_to(g_abi.effective_splits, abi, "bpt_effective_splits_scored");
  bind_to(g_abi.workspace_bytes, abi, "bpt_scored_workspace_bytes");
  bind_to(g_abi.decode, abi, "bpt_decode_scored");
  bind_to(g_abi.append, abi, "bpt_append_tokens");
  bind_to(g_abi.evict_moves, abi, "bpt_evict_moves");
  bind_to(g_abi.select, abi, "bpt_select_evictions");
  bind_to(g_abi.compact, abi, "bpt_compact_cache");
  g_argument_error = argument_error.inc_ref().ptr();
  g_check = check_fn.inc_ref().ptr();
}

}  // namespace

PYBIND11_MODULE(_bind, m) {
  m.def("init", &init);
  m.def("scored_workspace_bytes", &scored_workspace_bytes);
  m.def("decode_scored", &decode_scored);
  m.def("append_tokens", &append_tokens);
  m.def("select_evictions", &select_evictions);
  m.def("compact_cache", &compact_cache);
}
