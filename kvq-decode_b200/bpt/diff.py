"""Differential decode attention over a paged cache (no reference counterpart).

Two softmax maps with their own q and key heads are subtracted before they meet the values, so
that the attention which both give to irrelevant tokens cancels:

    o_j = (softmax(s q_2j . k_2h) - lam_j softmax(s q_2j+1 . k_2h+1)) v_h,   h = j // (H / Hkv)

for output heads j < H. q [B, 2 H, D]; k_cache [num_blocks, block_size, 2 Hkv, D]; v_cache
[num_blocks, block_size, Hkv, 2 D]; out [B, H, 2 D]. With a norm weight each head's output is
normalised by its root mean square, as such layers do; ``out_scale`` is their factor
1 - lambda_init.
"""
from typing import Optional

import torch

from .decode import _require
from .evict import _decode_scored


def diff_lambda(lambda_q1: torch.Tensor, lambda_k1: torch.Tensor, lambda_q2: torch.Tensor,
                lambda_k2: torch.Tensor, lambda_init: float, heads: int) -> torch.Tensor:
    """The layer's learned vectors [D] (shared by the heads) or [H, D] -> lam [H] fp32:
    exp(q1 . k1) - exp(q2 . k2) + lambda_init. Weights do not change while serving: call it once
    when they are loaded."""
    vectors = (lambda_q1, lambda_k1, lambda_q2, lambda_k2)
    _require(all(v.shape == vectors[0].shape for v in vectors) and
             vectors[0].dim() in (1, 2) and
             (vectors[0].dim() == 1 or vectors[0].shape[0] == heads),
             "lambda vectors must be [D] or [heads, D] of one shape")
    q1, k1, q2, k2 = (v.detach().float() for v in vectors)
    lam = torch.exp((q1 * k1).sum(-1)) - torch.exp((q2 * k2).sum(-1)) + lambda_init
    return lam.expand(heads).contiguous()


def paged_decode_attention_diff(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                block_table: torch.Tensor, seq_lens: torch.Tensor,
                                lam: torch.Tensor, scale: Optional[float] = None,
                                num_splits: Optional[int] = None, *,
                                norm_weight: Optional[torch.Tensor] = None,
                                norm_eps: float = 1e-5, out_scale: float = 1.0,
                                scores: Optional[torch.Tensor] = None, decay: float = 1.0,
                                out: Optional[torch.Tensor] = None,
                                workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Differential GQA decode over an fp16 or bf16 paged cache -> [B, H, 2 D].

    D 64 or 128, at most 4 output heads per value head; keys must be finite. lam is fp32 [H], or
    [B, H] where it depends on the token. norm_weight fp32 [2 D]: o / sqrt(mean(o^2) + norm_eps) *
    norm_weight, zeros where the mean is 0 (norm_eps may be 0); the result is then multiplied by
    out_scale. Softmax, sums and the norm are fp32, rounded once. With ``scores`` [B, Hkv, T] fp32
    (``bpt.evict``), slot t of value head h gets

        scores[b, h, t] = decay * scores[b, h, t] + sum_j |map-1 weight - lam_j * map-2 weight|

    the sum over its output heads: the weight by which the token's value counts. An empty
    sequence gives zeros. No host synchronisation.
    """
    return _decode_scored(2, q, k_cache, v_cache, block_table, seq_lens, scale, num_splits, scores,
                          decay, out, workspace, lam, norm_weight, norm_eps, out_scale)


__all__ = ["paged_decode_attention_diff", "diff_lambda"]
