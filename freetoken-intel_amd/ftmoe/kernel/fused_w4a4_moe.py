"""Routed MXFP4 experts with MXFP4 activations: x quantised, w13 and its activation, ``h``
quantised, w2, and the experts' rows summed with their router weights -- what
:mod:`~ftmoe.moe.token_sort` and :mod:`~ftmoe.kernel.w4a4_linear` compute call by call,
enqueued by one call.  Beside :func:`ftmoe.kernel.fused_moe.fused_moe` (dense
banks) and the MXFP4 banks of :class:`~ftmoe.layer.MoeLayer` (wide activations)."""
from __future__ import annotations

import ctypes

import torch

from .. import _native as nat
from ..layout import row_stride, rows_of
from ..moe.token_sort import ID_DTYPES
from .w4a4_linear import _QBLOCK, mxfp4_of
from .w8a8_linear import activation_code, bias_of


def fused_w4a4_moe(
    hidden_states: torch.Tensor,
    w1_blocks: torch.Tensor,
    w1_scales: torch.Tensor,
    w2_blocks: torch.Tensor,
    w2_scales: torch.Tensor,
    topk_ids: torch.Tensor,
    topk_w: torch.Tensor,
    *,
    activation: str = "silu",
    swiglu_alpha: float = 1.702,
    swiglu_limit: float = 7.0,
    w1_bias: torch.Tensor | None = None,
    w2_bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """``hidden_states [T, H]``, w1 ``[E, 2I, H/32, 16]`` (gate||up) and w2
    ``[E, H, I/32, 16]`` with their scales ``[E, 2I, H/32]`` and ``[E, H, I/32]``,
    ``topk_ids [T, k]`` (an id outside [0, E): no expert) and ``topk_w [T, k]`` ->
    ``[T, H]``.  ``h`` is quantised from fp32 and the experts' rows stay in fp32, the result is
    rounded once; no host synchronisation."""
    x = hidden_states
    nat.require_gpu(x, "hidden_states")
    nat.require_same_device(x, (("w1_blocks", w1_blocks), ("w1_scales", w1_scales), ("w2_blocks", w2_blocks),
                                ("w2_scales", w2_scales), ("topk_ids", topk_ids), ("topk_w", topk_w),
                                ("w1_bias", w1_bias), ("w2_bias", w2_bias)))
    if x.dim() != 2 or topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0] or topk_ids.shape[1] == 0:
        raise ValueError(f"hidden_states must be [T, H] and topk_ids [T, k], got {tuple(x.shape)} and "
                         f"{tuple(topk_ids.shape)}")
    if topk_w.shape != topk_ids.shape:
        raise ValueError(f"topk_w must be {list(topk_ids.shape)}, got {tuple(topk_w.shape)}")
    if topk_ids.dtype not in ID_DTYPES:
        raise TypeError(f"topk_ids must be int32 or int64, got {topk_ids.dtype}")
    (T, H), k = x.shape, topk_ids.shape[1]
    dt, w_dt, act = nat.dtype_code(x.dtype), nat.dtype_code(topk_w.dtype), activation_code(activation)
    wa, sa = mxfp4_of(w1_blocks, w1_scales, 2, "w1")
    wb, sb = mxfp4_of(w2_blocks, w2_scales, 2, "w2")
    E, I2 = wa.shape[:2]
    if _QBLOCK * wa.shape[2] != H:
        raise ValueError(f"hidden_states' H={H} does not match w1_blocks' implied K={_QBLOCK * wa.shape[2]}")
    if not 1 <= E <= 512:
        raise ValueError(f"between 1 and 512 experts, got {E}")
    if I2 % 2 or I2 == 0:
        raise ValueError(f"w1 must have gate rows, then up rows, got {I2} rows")
    if wb.shape[0] != E or wb.shape[1] != H or _QBLOCK * wb.shape[2] != I2 // 2:
        raise ValueError(f"w2_blocks must be {[E, H, I2 // 2 // _QBLOCK, 16]} for {I2} rows of w1, got {tuple(wb.shape)}")
    ba, ba_dt = bias_of(w1_bias, wa.shape[:2], "w1_bias")
    bb, bb_dt = bias_of(w2_bias, wb.shape[:2], "w2_bias")
    out = torch.empty(T, H, dtype=x.dtype, device=x.device)
    if T == 0:
        return out
    x, ids, w = rows_of(x), topk_ids.contiguous(), topk_w.contiguous()
    L = nat.lib()
    need = L.ftm_w4a4_moe_workspace_bytes(T, k, E, H, I2 // 2)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    c = nat.FtmW4A4Moe(x.data_ptr(), ids.data_ptr(), w.data_ptr(), out.data_ptr(), wa.data_ptr(), sa.data_ptr(),
                       nat.ptr(ba), wb.data_ptr(), sb.data_ptr(), nat.ptr(bb), row_stride(x) * x.element_size(), T, k, E,
                       H, I2 // 2, dt, ID_DTYPES[ids.dtype], w_dt, ba_dt, bb_dt, act, swiglu_alpha, swiglu_limit)
    nat.launch("ftm_w4a4_moe_forward", L.ftm_w4a4_moe_forward, x, ctypes.byref(c), ws.data_ptr(), need)
    return out


__all__ = ["fused_w4a4_moe"]
