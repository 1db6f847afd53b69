"""Routed INT8 experts with int8 activations, as grouped calls: the pairs sorted
by expert, the tokens quantised once, w13 and its activation, ``h`` quantised,
w2, and the rows back in token order with their router weights.  Beside
:func:`ftmoe.kernel.fused_moe.fused_moe` (dense banks) and the INT8 banks of
:class:`~ftmoe.layer.MoeLayer` (wide activations)."""
from __future__ import annotations

import torch

from ..moe.token_sort import combine_tokens, sort_tokens
from .w8a8_linear import quantize_int8_token, w8a8_grouped_linear


def fused_w8a8_moe(
    hidden_states: torch.Tensor,
    w1: torch.Tensor,
    w1_scale: torch.Tensor,
    w2: torch.Tensor,
    w2_scale: torch.Tensor,
    topk_ids: torch.Tensor,
    topk_w: torch.Tensor,
    *,
    activation: str = "silu",
    swiglu_alpha: float = 1.702,
    swiglu_limit: float = 7.0,
    w1_bias: torch.Tensor | None = None,
    w2_bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """``hidden_states [T, H]``, ``w1 [E, 2I, H]`` (gate||up) and ``w2 [E, H, I]`` as int8
    codes (or packed int32, the banks of an INT8 checkpoint) with scales ``[E, 2I]`` and
    ``[E, H]``, ``topk_ids [T, k]`` (an id outside [0, E): no expert) and ``topk_w [T, k]``
    -> ``[T, H]``.  ``h`` and the experts' rows stay in fp32, the result is rounded once; no
    host synchronisation."""
    if hidden_states.dim() != 2 or topk_ids.dim() != 2 or topk_ids.shape[0] != hidden_states.shape[0]:
        raise ValueError(f"hidden_states must be [T, H] and topk_ids [T, k], got {tuple(hidden_states.shape)} and "
                         f"{tuple(topk_ids.shape)}")
    if tuple(topk_w.shape) != tuple(topk_ids.shape):
        raise ValueError(f"topk_w must be {list(topk_ids.shape)}, got {tuple(topk_w.shape)}")
    sort = sort_tokens(topk_ids, w1.shape[0])
    q, s = quantize_int8_token(hidden_states)
    h = w8a8_grouped_linear(q, s, sort.offsets, w1, w1_scale, row_index=sort.token_of_row, bias=w1_bias,
                            activation=activation, swiglu_alpha=swiglu_alpha, swiglu_limit=swiglu_limit,
                            out_dtype=torch.float32)
    q, s = quantize_int8_token(h)
    y = w8a8_grouped_linear(q, s, sort.offsets, w2, w2_scale, bias=w2_bias, out_dtype=torch.float32)
    return combine_tokens(y, topk_w, sort, out_dtype=hidden_states.dtype)


__all__ = ["fused_w8a8_moe"]
