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
notice; keys carry their rotary position from when they were written.

Without a host synchronisation the calls plan for the table's and the rows' width, not for
the lengths. Where the caller knows that no sequence is longer than n slots, views of that width
(``block_table[:, :ceil(n / block_size)]``, ``scores[:, :, :n]``) save workspace, splits and CTAs.

Sequences that share pages (a common prefix) can be decoded and scored together, but a sequence
that is appended to or evicted must own its pages alone. ``bpt.diff`` has the differential decode
over such a cache.
"""
import ctypes
import importlib
from typing import NamedTuple, Optional

import torch

from . import _lib
from . import decode as _decode
from .decode import check_device_flags

_BIND = None
_ABI = ("bpt_effective_splits_scored", "bpt_scored_workspace_bytes", "bpt_decode_scored",
        "bpt_append_tokens", "bpt_evict_moves", "bpt_select_evictions", "bpt_compact_cache")


def _bind():
    """The extension module ``bpt/_bind``, calling into the library that ``bpt._lib`` loaded."""
    global _BIND
    if _BIND is None:
        lib = _lib.lib()
        try:
            module = importlib.import_module("._bind", __package__)
        except ModuleNotFoundError as e:
            raise ImportError("bpt/_bind is not built; build it with `python "
                              "kvq-decode_b200/build.py` (there is no fallback)") from e
        except ImportError as e:
            raise ImportError(f"bpt/_bind does not load ({e}); rebuild it for this torch with "
                              "`python kvq-decode_b200/build.py`") from e
        module.init({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _ABI},
                    _lib.BptArgumentError, _lib.check)
        _BIND = module
    return _BIND


class EvictionMoves(NamedTuple):
    """What ``select_evictions`` decided: rows src -> dst (logical slots, int32 [B, Hkv, M],
    -1 past counts), counts [B, Hkv] and the lengths after the move, new_lens [B]."""
    src: torch.Tensor
    dst: torch.Tensor
    counts: torch.Tensor
    new_lens: torch.Tensor


def _status(like: torch.Tensor) -> Optional[torch.Tensor]:
    """A zeroed status word in checked mode."""
    return torch.zeros(4, dtype=torch.uint8, device=like.device) if _decode.CHECKS else None


def _decode_scored(maps, q, k_cache, v_cache, block_table, seq_lens, scale, num_splits, scores,
                   decay, out, workspace, lam=None, norm_weight=None, norm_eps=0.0,
                   out_scale=1.0):
    bind = _BIND or _bind()
    if not _decode.CHECKS:
        return bind.decode_scored(maps, q, k_cache, v_cache, block_table, seq_lens, scale,
                                  num_splits, scores, decay, out, workspace, lam, norm_weight,
                                  norm_eps, out_scale)
    need = bind.scored_workspace_bytes(maps, q, k_cache, block_table, num_splits or 0,
                                       scores is not None)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    word = workspace.view(-1).view(torch.uint8)[:4]
    word.zero_()
    out = bind.decode_scored(maps, q, k_cache, v_cache, block_table, seq_lens, scale, num_splits,
                             scores, decay, out, workspace, lam, norm_weight, norm_eps, out_scale)
    check_device_flags(word, "bpt_decode_scored")
    return out


def scored_workspace_bytes(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor,
                           num_splits: Optional[int] = None, *, maps: int = 1,
                           scored: bool = True) -> int:
    """Bytes of a ``workspace`` for a decode of these shapes (maps 2: the differential one). A
    workspace serves calls that follow one another on a stream, captured ones among them; two
    calls that may run at the same time need one each. A call given less allocates its own."""
    return _bind().scored_workspace_bytes(maps, q, k_cache, block_table, num_splits or 0, scored)


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
    if scores is None:
        raise _lib.BptArgumentError("scores must be a tensor")
    return _decode_scored(1, q, k_cache, v_cache, block_table, seq_lens, scale, num_splits, scores,
                          decay, out, workspace)


def append_tokens(k_cache: torch.Tensor, v_cache: torch.Tensor, k_new: torch.Tensor,
                  v_new: torch.Tensor, new_lens: torch.Tensor, seq_lens: torch.Tensor,
                  block_table: torch.Tensor, *, scores: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None,
                  next_pos: Optional[torch.Tensor] = None) -> None:
    """Write tokens t < new_lens[b] of k_new / v_new [B, S, heads, D] (fp16 or bf16, as the cache)
    into the slots seq_lens[b] + t of a paged cache, S = 1 for a decode step.

    scores of the new slots become 0 and positions next_pos[b] + t where those are given. The
    heads are those of each cache, so a differential cache (``bpt.diff``) is appended to with the
    same call. Tokens past the block table are not written, and new_lens are clamped to [0, S]
    (checked mode raises on both). seq_lens is not changed: the caller advances it, by no more than
    was written. Runs on the current stream, no host synchronisation.
    """
    status = _status(k_cache)
    (_BIND or _bind()).append_tokens(k_cache, v_cache, k_new, v_new, new_lens, seq_lens,
                                     block_table, scores, positions, next_pos, status)
    if status is not None:
        check_device_flags(status, "bpt_append_tokens")


def select_evictions(scores: torch.Tensor, positions: torch.Tensor, seq_lens: torch.Tensor,
                     next_pos: torch.Tensor, budget: int, *, recent: int = 0, sinks: int = 0,
                     moves: Optional[EvictionMoves] = None) -> EvictionMoves:
    """Choose the ``budget`` tokens that each kv head of each sequence keeps -> EvictionMoves.

    Lengths count as at most the rows' width T. A sequence of at most budget tokens keeps all.
    Otherwise the tokens of position < sinks or >= next_pos - recent are kept (recent + sinks <=
    budget), then those of the highest score, ties and NaN (below every number) by the lowest slot.
    The moves bring them to slots 0 .. budget - 1: the i-th evicted slot below budget takes the i-th
    kept slot from the end. Nothing is moved yet; ``compact_cache`` does that. ``moves`` reuses the
    tensors of an earlier result.
    """
    return EvictionMoves._make((_BIND or _bind()).select_evictions(
        scores, positions, seq_lens, next_pos, budget, recent, sinks, moves))


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
    status = _status(k_cache)
    (_BIND or _bind()).compact_cache(k_cache, v_cache, block_table, moves.src, moves.dst,
                                     moves.counts, scores, positions, status)
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
