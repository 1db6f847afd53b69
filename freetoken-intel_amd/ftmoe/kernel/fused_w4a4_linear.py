"""MXFP4 projections with the activations quantised to the same format on the way.
Beside :mod:`ftmoe.kernel.fused_mxfp4_linear`, which keeps the activations wide:
the same weights at the 4-bit matrix rate, with the rounding of x to 4 bits added."""
from __future__ import annotations

import torch

from .w4a4_linear import _product


def fused_w4a4_linear(
    x: torch.Tensor,
    weight_blocks: torch.Tensor,
    weight_scales: torch.Tensor,
    *,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``quantize_mxfp4(x)`` times the weight (``weight_blocks [N, K/32, 16]``,
    ``weight_scales [N, K/32]``) ``(+ bias)``, in ``out_dtype`` (default: x's)."""
    return _product(x, None, weight_blocks, weight_scales, bias=bias,
                    out_dtype=out_dtype if out_dtype is not None else x.dtype)


def fused_w4a4_expert_forward(
    x: torch.Tensor,
    blocks_gate_up: torch.Tensor,
    scales_gate_up: torch.Tensor,
    blocks_down: torch.Tensor,
    scales_down: torch.Tensor,
    *,
    intermediate: int,
    activation: str = "silu",
    swiglu_alpha: float = 1.702,
    swiglu_limit: float = 7.0,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """One expert: ``down(act(gate(x)) * up(x))``, x and ``h`` each quantised (``h`` from fp32)."""
    if blocks_gate_up.shape[0] != 2 * intermediate:
        raise ValueError(f"blocks_gate_up must have {2 * intermediate} rows, got {blocks_gate_up.shape[0]}")
    h = _product(x, None, blocks_gate_up, scales_gate_up, bias=None, activation=activation, alpha=swiglu_alpha,
                 limit=swiglu_limit, out_dtype=torch.float32)
    return _product(h, None, blocks_down, scales_down, bias=None,
                    out_dtype=out_dtype if out_dtype is not None else x.dtype)


__all__ = ["fused_w4a4_linear", "fused_w4a4_expert_forward"]
