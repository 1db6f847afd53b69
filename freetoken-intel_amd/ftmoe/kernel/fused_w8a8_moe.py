"""Routed INT8 experts with int8 activations, as grouped calls: the pairs sorted
by expert, the tokens quantised once, w13 and its activation, ``h`` quantised,
w2, and the rows back in token order with their router weights -- the bits of
:mod:`~ftmoe.moe.token_sort` and :mod:`~ftmoe.kernel.w8a8_linear` called one by
one, enqueued by one call.  Beside
:func:`ftmoe.kernel.fused_moe.fused_moe` (dense banks) and the INT8 banks of
:class:`~ftmoe.layer.MoeLayer` (wide activations)."""
from __future__ import annotations

import ctypes

import torch

from .. import _native as nat
from ..layout import row_stride, rows_of
from ..moe.token_sort import ID_DTYPES
from .w8a8_linear import activation_code, bias_of, scale_of, weight_of


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
    x = hidden_states
    nat.require_gpu(x, "hidden_states")
    nat.require_same_device(x, (("w1", w1), ("w1_scale", w1_scale), ("w2", w2), ("w2_scale", w2_scale),
                                ("topk_ids", topk_ids), ("topk_w", topk_w), ("w1_bias", w1_bias), ("w2_bias", w2_bias)))
    if x.dim() != 2 or topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0] or topk_ids.shape[1] == 0:
        raise ValueError(f"hidden_states must be [T, H] and topk_ids [T, k], got {tuple(x.shape)} and "
                         f"{tuple(topk_ids.shape)}")
    if topk_w.shape != topk_ids.shape:
        raise ValueError(f"topk_w must be {list(topk_ids.shape)}, got {tuple(topk_w.shape)}")
    if topk_ids.dtype not in ID_DTYPES:
        raise TypeError(f"topk_ids must be int32 or int64, got {topk_ids.dtype}")
    (T, H), k = x.shape, topk_ids.shape[1]
    dt, w_dt, act = nat.dtype_code(x.dtype), nat.dtype_code(topk_w.dtype), activation_code(activation)
    wa, packed_a = weight_of(w1, H, 3, "w1")
    E, I2 = wa.shape[:2]
    if not 1 <= E <= 512:
        raise ValueError(f"between 1 and 512 experts, got {E}")
    if I2 % 2 or I2 == 0:
        raise ValueError(f"w1 must have gate rows, then up rows, got {I2} rows")
    wb, packed_b = weight_of(w2, I2 // 2, 3, "w2")
    if wb.shape[0] != E or wb.shape[1] != H:
        raise ValueError(f"w2 must be {[E, H, I2 // 2]}, got {[*wb.shape[:2], I2 // 2]}")
    sa, sa_dt = scale_of(w1_scale, wa.shape[:2], "w1_scale")
    sb, sb_dt = scale_of(w2_scale, wb.shape[:2], "w2_scale")
    ba, ba_dt = bias_of(w1_bias, wa.shape[:2], "w1_bias")
    bb, bb_dt = bias_of(w2_bias, wb.shape[:2], "w2_bias")
    out = torch.empty((T, H), dtype=x.dtype, device=x.device)
    if T == 0:
        return out
    x, ids, w = rows_of(x), topk_ids.contiguous(), topk_w.contiguous()
    L = nat.lib()
    need = L.ftm_w8a8_moe_workspace_bytes(T, k, E, H, I2 // 2)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    c = nat.FtmW8A8Moe(x.data_ptr(), ids.data_ptr(), w.data_ptr(), out.data_ptr(), wa.data_ptr(), sa.data_ptr(),
                       nat.ptr(ba), wb.data_ptr(), sb.data_ptr(), nat.ptr(bb), row_stride(x) * x.element_size(), T, k, E,
                       H, I2 // 2, dt, ID_DTYPES[ids.dtype], w_dt, packed_a, packed_b, sa_dt, ba_dt, sb_dt, bb_dt, act,
                       swiglu_alpha, swiglu_limit)
    nat.launch("ftm_w8a8_moe_forward", L.ftm_w8a8_moe_forward, x, ctypes.byref(c), ws.data_ptr(), need)
    return out


__all__ = ["fused_w8a8_moe"]
