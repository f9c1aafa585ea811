"""Bounded KV caches: decode attention that scores the cached tokens, and the eviction of those
that attention does not use (no reference counterpart).

The cache is the 16-bit paged cache of ``bpt.paged_decode_attention`` (fp16 here, or bf16). Beside
it the caller keeps, for every (sequence, kv head, logical slot),

    scores    [B, Hkv, T] fp32    the attention weight that the slot's token has received
    positions [B, Hkv, T] int32   the token's position in its sequence

with T at least the slots of a sequence (max_blocks * block_size), unit inner stride. A decode
step is

    append_tokens(k_cache, v_cache, k_new, v_new, new_lens, seq_lens, block_table,
                  scores=scores, positions=positions, next_pos=next_pos)
    seq_lens += new_lens; next_pos += new_lens
    out = paged_decode_attention_scored(q, k_cache, v_cache, block_table, seq_lens, scores)

and, when a sequence has grown past its budget (all layers have their own state),

    seq_lens = evict_tokens(k_cache, v_cache, block_table, seq_lens, scores, positions, next_pos,
                            budget, recent=..., sinks=...)

after which every sequence has at most ``budget`` tokens, in slots 0 .. new_len - 1: the pages
past them are free. Evicted caches hold their tokens out of order, which attention does not
notice; keys carry their rotary position from when they were written. Sequences that share
pages (a common prefix) can be decoded and scored together, but a sequence that is appended to
or evicted must own its pages alone. ``bpt.diff`` has the differential decode over such a cache.
"""
import ctypes
import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from .decode import _pow2, _require, _sm_count, _stream_handle, check_device_flags
from . import decode as _decode

c_i32, c_i64, c_f32, c_vp, c_size = (ctypes.c_int, ctypes.c_int64, ctypes.c_float,
                                     ctypes.c_void_p, ctypes.c_size_t)
DTYPES = {torch.float16: 1, torch.bfloat16: 2}


class ScoredDecodeC(ctypes.Structure):
    """Mirror of ``bpt_scored_decode`` (include/bpt.h)."""
    _fields_ = [("dtype", c_i32), ("maps", c_i32), ("batch", c_i32), ("q_heads", c_i32),
                ("kv_heads", c_i32), ("head_dim", c_i32), ("block_size", c_i32),
                ("max_blocks", c_i32), ("num_splits", c_i32), ("sm_count", c_i32),
                ("scale", c_f32), ("decay", c_f32), ("norm_eps", c_f32), ("out_scale", c_f32),
                ("num_blocks", c_i64), ("q", c_vp), ("q_stride", c_i64 * 2),
                ("k_cache", c_vp), ("k_stride", c_i64 * 3),
                ("v_cache", c_vp), ("v_stride", c_i64 * 3),
                ("block_table", c_vp), ("bt_stride", c_i64), ("seq_lens", c_vp),
                ("out", c_vp), ("out_stride", c_i64 * 2),
                ("scores", c_vp), ("scores_stride", c_i64 * 2),
                ("lam", c_vp), ("lam_stride", c_i64 * 2), ("norm_weight", c_vp)]


class PagedCacheC(ctypes.Structure):
    """Mirror of ``bpt_paged_cache`` (include/bpt.h)."""
    _fields_ = [("block_size", c_i32), ("k_heads", c_i32), ("v_heads", c_i32), ("k_dim", c_i32),
                ("v_dim", c_i32), ("num_blocks", c_i64), ("k", c_vp), ("k_stride", c_i64 * 3),
                ("v", c_vp), ("v_stride", c_i64 * 3)]


class EvictionMoves(NamedTuple):
    """What ``select_evictions`` decided: rows src -> dst (logical slots, int32 [B, Hkv, M],
    -1 past counts), counts [B, Hkv] and the lengths after the move, new_lens [B]."""
    src: torch.Tensor
    dst: torch.Tensor
    counts: torch.Tensor
    new_lens: torch.Tensor


_FNS = {}


def _fn(name):
    if not _FNS:
        P, C = ctypes.POINTER(ScoredDecodeC), ctypes.POINTER(PagedCacheC)
        strides = ctypes.POINTER(c_i64)
        state = [c_vp, c_i64, c_i64, c_vp, c_i64, c_i64]
        for n, res, args in (
                ("bpt_effective_splits_scored", c_i32, [c_i32] * 8),
                ("bpt_scored_workspace_bytes", c_size, [c_i32] * 5 + [c_i64]),
                ("bpt_decode_scored", c_i32, [P, c_vp, c_size, c_vp]),
                ("bpt_append_tokens", c_i32,
                 [C, c_vp, strides, c_vp, strides, c_vp, c_vp, c_vp, c_i64, c_i32, c_i32, c_i32] +
                 state + [c_vp, c_vp, c_vp]),
                ("bpt_evict_moves", c_i32, [c_i32, c_i32]),
                ("bpt_select_evictions", c_i32,
                 state + [c_vp, c_vp] + [c_i32] * 6 + [c_vp] * 5),
                ("bpt_compact_cache", c_i32,
                 [C, c_vp, c_i64, c_i32, c_vp, c_vp, c_vp, c_i32, c_i32] + state +
                 [c_i32, c_vp, c_vp])):
            _FNS[n] = _lib.register(n, res, args)
    return _FNS[name]


def _on(device, **tensors):
    for name, t in tensors.items():
        if t is not None:
            _require(t.device == device, f"{name} is on {t.device}, not on {device}")


def _check_cache(k_cache, v_cache, maps=1):
    """Shapes of a 16-bit paged cache: (dtype code, block_size, kv heads, v row width)."""
    _require(k_cache.dim() == 4 and v_cache.dim() == 4 and
             k_cache.shape[:2] == v_cache.shape[:2],
             "k_cache/v_cache must be [num_blocks, block_size, heads, D] of the same pages")
    _require(k_cache.dtype == v_cache.dtype and k_cache.dtype in DTYPES,
             "k_cache and v_cache must both be float16 or both bfloat16")
    _require(k_cache.stride(3) == 1 and v_cache.stride(3) == 1,
             "innermost (head_dim) stride must be 1")
    _require(_pow2(k_cache.shape[1]) and k_cache.shape[1] >= 16,
             "block_size must be a power of two >= 16")
    _require(k_cache.shape[2] == maps * v_cache.shape[2],
             f"k_cache must have {maps} heads for each head of v_cache")
    _require(k_cache.device.type == "cuda", "bpt runs on CUDA tensors only (no CPU fallback)")
    return DTYPES[k_cache.dtype], k_cache.shape[1], v_cache.shape[2], v_cache.shape[3]


def _check_rows(block_table, lens, B, names=("seq_lens",)):
    _require(block_table.dim() == 2 and block_table.shape[0] == B and
             block_table.dtype == torch.int32 and
             (block_table.stride(1) == 1 or block_table.shape[1] <= 1),
             "block_table must be int32 [B, max_blocks] with contiguous rows")
    for t, name in zip(lens, names):
        _require(t.shape == (B,) and t.dtype == torch.int32 and t.is_contiguous(),
                 f"{name} must be contiguous int32 [B]")


def _check_state(t, name, dtype, B, H, slots):
    _require(t.dim() == 3 and t.shape[0] == B and t.shape[1] == H and t.dtype == dtype and
             t.shape[2] >= slots and (t.stride(2) == 1 or t.shape[2] <= 1),
             f"{name} must be {str(dtype)[6:]} [{B}, {H}, >= {slots}] with a unit inner stride")


def _no_overlap(t, name):
    """Tensors that are written: no dimension may revisit the same memory."""
    _require(all(st != 0 or n <= 1 for n, st in zip(t.shape, t.stride())),
             f"{name} is written and cannot be an expanded view")


def _state_args(t):
    return (t.data_ptr(), t.stride(0), t.stride(1)) if t is not None else (None, 0, 0)


def _decode_scored(maps, q, k_cache, v_cache, block_table, seq_lens, scale, num_splits, scores,
                   decay, out, workspace, lam=None, norm_weight=None, norm_eps=0.0,
                   out_scale=1.0):
    _require(q.dim() == 3 and q.stride(2) == 1, "q must be [B, heads, D] with a unit inner stride")
    dt, bs, H, width = _check_cache(k_cache, v_cache, maps)
    B, Hq, D = q.shape
    dev = q.device
    _require(q.dtype == k_cache.dtype, "q and the caches must have the same dtype")
    _require(k_cache.shape[3] == D and width == maps * D,
             "head_dim of q and the caches do not match")
    _require(Hq % (maps * H) == 0, "q heads must be a multiple of the key heads")
    _check_rows(block_table, (seq_lens,), B)
    max_blocks = block_table.shape[1]
    cap = max_blocks * bs
    if scores is not None:
        _check_state(scores, "scores", torch.float32, B, H, cap)
        _no_overlap(scores, "scores")
    _on(dev, k_cache=k_cache, v_cache=v_cache, block_table=block_table, seq_lens=seq_lens,
        scores=scores, lam=lam, norm_weight=norm_weight, out=out, workspace=workspace)
    _require(math.isfinite(decay) and decay >= 0.0, "decay must be finite and not negative")
    sms = _sm_count(dev.index or 0)
    ns = int(num_splits or 0)
    S = _fn("bpt_effective_splits_scored")(D, maps, B, H, bs, max_blocks, ns, sms)
    need = _fn("bpt_scored_workspace_bytes")(D, maps, B, Hq, S, cap if scores is not None else 0)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    else:
        _require(workspace.is_contiguous(), "workspace must be contiguous")
    if out is None:
        out = torch.empty(B, Hq // maps, width, dtype=q.dtype, device=dev)
    else:
        _require(out.shape == (B, Hq // maps, width) and out.dtype == q.dtype and
                 out.stride(2) == 1,
                 f"out must be {q.dtype} {(B, Hq // maps, width)} with a unit inner stride")
        _no_overlap(out, "out")
    a = ScoredDecodeC()
    a.dtype, a.maps, a.batch, a.q_heads, a.kv_heads, a.head_dim = dt, maps, B, Hq, H, D
    a.block_size, a.max_blocks, a.num_blocks = bs, max_blocks, k_cache.shape[0]
    a.num_splits, a.sm_count = ns, sms
    a.scale = 0.0 if scale is None else scale
    a.decay, a.norm_eps, a.out_scale = decay, norm_eps, out_scale
    a.q, a.q_stride[:] = q.data_ptr(), q.stride()[:2]
    a.k_cache, a.k_stride[:] = k_cache.data_ptr(), k_cache.stride()[:3]
    a.v_cache, a.v_stride[:] = v_cache.data_ptr(), v_cache.stride()[:3]
    a.block_table, a.bt_stride = block_table.data_ptr(), block_table.stride(0)
    a.seq_lens = seq_lens.data_ptr()
    a.out, a.out_stride[:] = out.data_ptr(), out.stride()[:2]
    if scores is not None:
        a.scores, a.scores_stride[:] = scores.data_ptr(), scores.stride()[:2]
    if lam is not None:
        a.lam = lam.data_ptr()
        a.lam_stride[:] = (lam.stride(0) if lam.dim() == 2 else 0, lam.stride(-1))
    if norm_weight is not None:
        a.norm_weight = norm_weight.data_ptr()
    if _decode.CHECKS:
        workspace.view(-1).view(torch.uint8)[:4].zero_()
    with torch.cuda.device(dev):
        rc = _fn("bpt_decode_scored")(ctypes.byref(a), workspace.data_ptr(),
                                      workspace.numel() * workspace.element_size(),
                                      _stream_handle(dev))
    _lib.check(rc, "bpt_decode_scored")
    if _decode.CHECKS:
        check_device_flags(workspace.view(-1).view(torch.uint8), "bpt_decode_scored")
    return out


def scored_workspace_bytes(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor,
                           num_splits: Optional[int] = None, *, maps: int = 1,
                           scored: bool = True) -> int:
    """Bytes of a ``workspace`` for a decode of these shapes (maps 2: the differential one). A
    workspace serves calls that follow one another on a stream, captured ones among them; two
    calls that may run at the same time need one each."""
    B, Hq, D = q.shape
    bs, H, mb = k_cache.shape[1], k_cache.shape[2] // maps, block_table.shape[1]
    S = _fn("bpt_effective_splits_scored")(D, maps, B, H, bs, mb, int(num_splits or 0),
                                           _sm_count(q.device.index or 0))
    return int(_fn("bpt_scored_workspace_bytes")(D, maps, B, Hq, S, mb * bs if scored else 0))


def paged_decode_attention_scored(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                  block_table: torch.Tensor, seq_lens: torch.Tensor,
                                  scores: torch.Tensor, scale: Optional[float] = None,
                                  num_splits: Optional[int] = None, *, decay: float = 1.0,
                                  out: Optional[torch.Tensor] = None,
                                  workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """GQA decode over an fp16 or bf16 paged cache -> [B, Hq, D], scoring the cached tokens.

    As ``bpt.paged_decode_attention`` (layout, split semantics, no host synchronisation, zeros
    for an empty sequence), for head_dim 64, 128 or 256 and at most 8 q heads per kv head. Slot t
    of kv head h of sequence b, t < seq_lens[b], gets

        scores[b, h, t] = decay * scores[b, h, t] + sum over the head's q heads of softmax weight t

    in place, in fp32. decay 1 accumulates, less than 1 fades, 0 keeps this step's weights only
    (the old scores are not read). Slots past seq_lens[b] keep their scores.
    """
    _require(scores is not None, "scores must be a tensor")
    return _decode_scored(1, q, k_cache, v_cache, block_table, seq_lens, scale, num_splits, scores,
                          float(decay), out, workspace)


def _cache_c(k_cache, v_cache, bs):
    c = PagedCacheC()
    c.block_size, c.num_blocks = bs, k_cache.shape[0]
    c.k_heads, c.k_dim = k_cache.shape[2:]
    c.v_heads, c.v_dim = v_cache.shape[2:]
    c.k, c.k_stride[:] = k_cache.data_ptr(), k_cache.stride()[:3]
    c.v, c.v_stride[:] = v_cache.data_ptr(), v_cache.stride()[:3]
    return c


def _status(dev):
    return torch.zeros(4, dtype=torch.uint8, device=dev) if _decode.CHECKS else None


def append_tokens(k_cache: torch.Tensor, v_cache: torch.Tensor, k_new: torch.Tensor,
                  v_new: torch.Tensor, new_lens: torch.Tensor, seq_lens: torch.Tensor,
                  block_table: torch.Tensor, *, scores: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None,
                  next_pos: Optional[torch.Tensor] = None) -> None:
    """Write tokens t < new_lens[b] of k_new / v_new [B, S, heads, D] (fp16 or bf16, as the cache)
    into the slots seq_lens[b] + t of a paged cache, S = 1 for a decode step.

    scores of the new slots become 0 and positions next_pos[b] + t where those are given. The
    heads are those of each cache, so a differential cache (``bpt.diff``) is appended to with the
    same call. Tokens past the block table are not written (checked mode raises). seq_lens
    is not changed: the caller advances it. Runs on the current stream, no host synchronisation.
    """
    _require(v_cache.dim() == 4 and k_cache.dim() == 4 and v_cache.shape[2] > 0,
             "k_cache/v_cache must be [num_blocks, block_size, heads, D]")
    _, bs, H, _ = _check_cache(k_cache, v_cache, max(1, k_cache.shape[2] // v_cache.shape[2]))
    dev = k_cache.device
    _require(k_new.dim() == 4 and v_new.dim() == 4 and k_new.shape[:2] == v_new.shape[:2] and
             k_new.shape[2:] == k_cache.shape[2:] and v_new.shape[2:] == v_cache.shape[2:],
             "k_new/v_new must be [B, S, heads, D] with the heads and widths of their caches")
    _require(k_new.dtype == v_new.dtype == k_cache.dtype, "k_new/v_new must have the cache's dtype")
    _require(k_new.stride(3) == 1 and v_new.stride(3) == 1, "k_new/v_new need a unit inner stride")
    B, S = k_new.shape[:2]
    _check_rows(block_table, (new_lens, seq_lens), B, ("new_lens", "seq_lens"))
    cap = block_table.shape[1] * bs
    for t, name, want in ((scores, "scores", torch.float32), (positions, "positions", torch.int32)):
        if t is not None:
            _check_state(t, name, want, B, H, cap)
            _no_overlap(t, name)
    _require(positions is None or next_pos is not None, "positions need next_pos")
    if next_pos is not None:
        _check_rows(block_table, (next_pos,), B, ("next_pos",))
    _no_overlap(k_cache, "k_cache")
    _no_overlap(v_cache, "v_cache")
    _on(dev, v_cache=v_cache, k_new=k_new, v_new=v_new, new_lens=new_lens, seq_lens=seq_lens,
        block_table=block_table, scores=scores, positions=positions, next_pos=next_pos)
    c = _cache_c(k_cache, v_cache, bs)
    status = _status(dev)
    with torch.cuda.device(dev):
        rc = _fn("bpt_append_tokens")(
            ctypes.byref(c), k_new.data_ptr(), (c_i64 * 3)(*k_new.stride()[:3]),
            v_new.data_ptr(), (c_i64 * 3)(*v_new.stride()[:3]), new_lens.data_ptr(),
            seq_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0),
            block_table.shape[1], B, S, *_state_args(scores), *_state_args(positions),
            next_pos.data_ptr() if next_pos is not None else None,
            status.data_ptr() if status is not None else None, _stream_handle(dev))
    _lib.check(rc, "bpt_append_tokens")
    if status is not None:
        check_device_flags(status, "bpt_append_tokens")


def select_evictions(scores: torch.Tensor, positions: torch.Tensor, seq_lens: torch.Tensor,
                     next_pos: torch.Tensor, budget: int, *, recent: int = 0, sinks: int = 0,
                     moves: Optional[EvictionMoves] = None) -> EvictionMoves:
    """Choose the ``budget`` tokens that each kv head of each sequence keeps -> EvictionMoves.

    A sequence of at most budget tokens keeps all. Otherwise the tokens of position < sinks or
    >= next_pos - recent are kept (recent + sinks <= budget), then those of the highest score,
    ties and NaN (below every number) by the lowest slot. The moves bring them to slots 0 ..
    budget - 1: the i-th evicted slot below budget takes the i-th kept slot from the end. Nothing is
    moved yet; ``compact_cache`` does that. ``moves`` reuses the tensors of an earlier result.
    """
    _require(scores.dim() == 3 and positions.shape == scores.shape,
             "scores and positions must be [B, Hkv, T]")
    B, H, T = scores.shape
    _check_state(scores, "scores", torch.float32, B, H, 0)
    _check_state(positions, "positions", torch.int32, B, H, 0)
    for t, name in ((seq_lens, "seq_lens"), (next_pos, "next_pos")):
        _require(t.shape == (B,) and t.dtype == torch.int32 and t.is_contiguous(),
                 f"{name} must be contiguous int32 [B]")
    dev = scores.device
    _require(dev.type == "cuda", "bpt runs on CUDA tensors only (no CPU fallback)")
    _require(budget >= 1 and recent >= 0 and sinks >= 0 and recent + sinks <= budget,
             "budget must be at least 1 and at least recent + sinks")
    _require(budget < 1 << 31, "budget must be an int32")
    M = _fn("bpt_evict_moves")(budget, T)
    if moves is None:
        pair = torch.empty(2, B, H, M, dtype=torch.int32, device=dev)
        moves = EvictionMoves(pair[0], pair[1],
                              torch.empty(B, H, dtype=torch.int32, device=dev),
                              torch.empty(B, dtype=torch.int32, device=dev))
    else:
        for t, shape in zip(moves, ((B, H, M), (B, H, M), (B, H), (B,))):
            _require(t.shape == shape and t.dtype == torch.int32 and t.is_contiguous(),
                     f"moves must be contiguous int32 tensors {(B, H, M)} x 2, {(B, H)}, {(B,)}")
    _require(moves.new_lens.data_ptr() != seq_lens.data_ptr() or B == 0,
             "moves.new_lens cannot be seq_lens itself")
    _on(dev, positions=positions, seq_lens=seq_lens, next_pos=next_pos, **moves._asdict())
    with torch.cuda.device(dev):
        rc = _fn("bpt_select_evictions")(
            *_state_args(scores), *_state_args(positions), seq_lens.data_ptr(),
            next_pos.data_ptr(), B, H, T, budget, recent, sinks, moves.src.data_ptr(),
            moves.dst.data_ptr(), moves.counts.data_ptr(), moves.new_lens.data_ptr(),
            _stream_handle(dev))
    _lib.check(rc, "bpt_select_evictions")
    return moves


def compact_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  moves: EvictionMoves, scores: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None) -> None:
    """Carry out ``moves`` in place: rows src -> dst of k_cache, v_cache and, where given, of
    scores and positions (give them whenever the cache is evicted again).

    The caches [num_blocks, block_size, Hkv, D] may have different widths D (multiples of 8). A
    differential cache's pairs of key heads move as one head: pass
    ``k_cache.view(num_blocks, block_size, Hkv, 2 * D)``. Rows that no move names keep their
    contents, slots past the new length included. Invalid moves are skipped (checked mode raises).
    """
    _, bs, H, _ = _check_cache(k_cache, v_cache)
    dev = k_cache.device
    src, dst, counts, _new = moves
    _require(src.dim() == 3 and src.shape[1] == H and src.shape == dst.shape and
             counts.shape == src.shape[:2], "moves must be src/dst [B, Hkv, M], counts [B, Hkv]")
    B, _, M = src.shape
    for t, name in ((src, "src"), (dst, "dst"), (counts, "counts")):
        _require(t.dtype == torch.int32 and t.is_contiguous(),
                 f"moves.{name} must be contiguous int32")
    _check_rows(block_table, (), B)
    slots = block_table.shape[1] * bs
    for t, name, want in ((scores, "scores", torch.float32), (positions, "positions", torch.int32)):
        if t is not None:
            _check_state(t, name, want, B, H, 0)
            _no_overlap(t, name)
            slots = min(slots, t.shape[2])
    _no_overlap(k_cache, "k_cache")
    _no_overlap(v_cache, "v_cache")
    _on(dev, v_cache=v_cache, block_table=block_table, scores=scores, positions=positions,
        src=src, dst=dst, counts=counts)
    c = _cache_c(k_cache, v_cache, bs)
    status = _status(dev)
    with torch.cuda.device(dev):
        rc = _fn("bpt_compact_cache")(
            ctypes.byref(c), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            src.data_ptr(), dst.data_ptr(), counts.data_ptr(), M, B, *_state_args(scores),
            *_state_args(positions), slots,
            status.data_ptr() if status is not None else None, _stream_handle(dev))
    _lib.check(rc, "bpt_compact_cache")
    if status is not None:
        check_device_flags(status, "bpt_compact_cache")


def evict_tokens(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, scores: torch.Tensor, positions: torch.Tensor,
                 next_pos: torch.Tensor, budget: int, *, recent: int = 0, sinks: int = 0,
                 moves: Optional[EvictionMoves] = None) -> torch.Tensor:
    """``select_evictions`` and ``compact_cache``: bring every sequence down to ``budget`` tokens.
    Returns the new lengths [B] int32 (seq_lens itself is not changed)."""
    m = select_evictions(scores, positions, seq_lens, next_pos, budget, recent=recent,
                         sinks=sinks, moves=moves)
    compact_cache(k_cache, v_cache, block_table, m, scores, positions)
    return m.new_lens


__all__ = ["paged_decode_attention_scored", "scored_workspace_bytes", "append_tokens",
           "select_evictions", "compact_cache", "evict_tokens", "EvictionMoves"]
