"""INT8 projections with the activations quantised on the way: one scale per
token, found at run time.  Beside :mod:`ftmoe.kernel.fused_int8_linear`, which
keeps the activations wide: the same weights at the int8 matrix rate, with the
rounding of x to 8 bits (half a step of max |x| / 127 at most) added."""
from __future__ import annotations

import torch

from .w8a8_linear import _product


def fused_w8a8_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    *,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``quantize_int8_token(x)`` times ``weight`` (int8 ``[N, K]`` or packed int32
    ``[N, K/4]``, ``weight_scale [N]``) ``(+ bias)``, in ``out_dtype`` (default: x's)."""
    return _product(x, None, weight, weight_scale, bias=bias, out_dtype=out_dtype if out_dtype is not None else x.dtype)


def fused_w8a8_expert_forward(
    x: torch.Tensor,
    weight_gate_up: torch.Tensor,
    weight_scale_gate_up: torch.Tensor,
    weight_down: torch.Tensor,
    weight_scale_down: torch.Tensor,
    *,
    intermediate: int,
    activation: str = "silu",
    swiglu_alpha: float = 1.702,
    swiglu_limit: float = 7.0,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """One expert: ``down(act(gate(x)) * up(x))``, x and ``h`` each quantised by token
    (``h`` from fp32)."""
    if weight_gate_up.shape[0] != 2 * intermediate:
        raise ValueError(f"weight_gate_up must have {2 * intermediate} rows, got {weight_gate_up.shape[0]}")
    h = _product(x, None, weight_gate_up, weight_scale_gate_up, bias=None, activation=activation,
                 alpha=swiglu_alpha, limit=swiglu_limit, out_dtype=torch.float32)
    return _product(h, None, weight_down, weight_scale_down, bias=None,
                    out_dtype=out_dtype if out_dtype is not None else x.dtype)


__all__ = ["fused_w8a8_linear", "fused_w8a8_expert_forward"]
