"""Int8 activations x int8 weights: the per-token quantiser and the integer
product with one scale per token and one per output channel, dense or grouped
by expert.  The reference has INT8 weights under wide activations only
(python/freetoken/kernel/triton/fused_int8_linear.py); the weights here are the
same codes and scales, either plain int8 ``[N, K]``
(:func:`~ftmoe.quant.quantize_int8_channel`) or the checkpoint's packed int32
``[N, K/4]`` (offset-binary bytes, one scale a row).

gfx950: int32 sums on the int8 matrix cores, exact for K up to 131071, so a
result does not depend on the batch it is computed in; scales, bias and the
gated activation are applied in fp32 in the same kernel and rounded once."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .. import _native as nat
from ..layer import ACTIVATIONS

_SCALE_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def quantize_int8_token(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [..., K]`` (fp32, fp16 or bf16) -> (int8 codes ``[..., K]``, fp32 scales
    ``[...]``): scale = max |x| / 127 of the row (the maximum at least 1e-12), code
    = the whole number nearest x / scale, ties to even.  A row with an infinity or
    NaN gets the scale NaN and codes 0: its products are NaN, no other row's are."""
    nat.require_gpu(x, "x")
    dt = nat.dtype_code(x.dtype)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., K] with K > 0, got {tuple(x.shape)}")
    lead, K = x.shape[:-1], x.shape[-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if x2.stride(1) != 1 and K > 1:
        x2 = x2.contiguous()
    rows = x2.shape[0]
    q = torch.empty((*lead, K), dtype=torch.int8, device=x.device)
    scale = torch.empty(lead, dtype=torch.float32, device=x.device)
    if rows == 0:
        return q, scale
    with nat.on_device_of(x):
        rc = nat.lib().ftm_quant_int8(x2.data_ptr(), dt, rows, K, x2.stride(0) * x2.element_size(), q.data_ptr(), K,
                                      scale.data_ptr(), nat.stream_of(x))
    nat.check(rc, "ftm_quant_int8")
    return q, scale


def _weight(weight: torch.Tensor, K: int, dim: int) -> tuple[torch.Tensor, int]:
    """(contiguous weight, packed) after the checks the formats share."""
    if weight.dtype not in (torch.int8, torch.int32):
        raise TypeError(f"weight must be int8 or packed int32, got {weight.dtype}")
    if weight.dim() != dim:
        raise ValueError(f"weight must have {dim} dimensions, got shape {tuple(weight.shape)}")
    packed = weight.dtype == torch.int32
    k = weight.shape[-1] * (4 if packed else 1)
    if k != K:
        raise ValueError(f"x's K={K} does not match the weight's K={k}")
    if K > nat.W8A8_MAX_K:
        raise ValueError(f"K={K} exceeds {nat.W8A8_MAX_K}: int32 sums of int8 products could overflow")
    return weight.contiguous(), int(packed)


def _per_channel(t: torch.Tensor, shape: tuple, name: str) -> torch.Tensor:
    if t.dtype not in _SCALE_DTYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if tuple(t.shape) != shape and (name != "weight_scale" or tuple(t.shape) != (*shape, 1)):
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    return t.contiguous()


def _product(x_int8, x_scale, weight, weight_scale, *, offsets, row_index, bias, activation, swiglu_alpha,
             swiglu_limit, out_dtype) -> torch.Tensor:
    nat.require_gpu(x_int8, "x_int8")
    nat.require_same_device(x_int8, (("x_scale", x_scale), ("weight", weight), ("weight_scale", weight_scale),
                                     ("bias", bias), ("offsets", offsets), ("row_index", row_index)))
    if x_int8.dtype != torch.int8:
        raise TypeError(f"x_int8 must be int8, got {x_int8.dtype}")
    if x_int8.dim() != 2 or x_int8.shape[1] == 0:
        raise ValueError(f"x_int8 must be [M, K] with K > 0, got {tuple(x_int8.shape)}")
    M, K = x_int8.shape
    if x_scale.dtype != torch.float32:
        raise TypeError(f"x_scale must be float32, got {x_scale.dtype}")
    if tuple(x_scale.shape) not in ((M,), (M, 1)):
        raise ValueError(f"x_scale must be [{M}], got {tuple(x_scale.shape)}")
    w, packed = _weight(weight, K, 2 if offsets is None else 3)
    N = w.shape[-2]
    ws = _per_channel(weight_scale, tuple(w.shape[:-1]), "weight_scale")
    b = _per_channel(bias, tuple(w.shape[:-1]), "bias") if bias is not None else None
    act = -1
    if activation is not None:
        if activation not in ACTIVATIONS:
            raise ValueError(f"unsupported MoE activation: {activation!r}")
        if N % 2:
            raise ValueError(f"a gated activation needs an even number of weight rows (gate, then up), got {N}")
        act = ACTIVATIONS[activation]
    if x_int8.stride(1) != 1 and K > 1:
        x_int8 = x_int8.contiguous()
    x_scale = x_scale.contiguous()
    rows = M if row_index is None else row_index.shape[0]
    out = torch.empty((rows, N // 2 if act >= 0 else N), dtype=out_dtype, device=x_int8.device)
    if out.numel() == 0:
        return out
    if M == 0:  # an index into no rows
        return out.zero_()
    c = nat.FtmW8A8(x_int8.data_ptr(), x_scale.data_ptr(), w.data_ptr(), ws.data_ptr(), nat.ptr(b), out.data_ptr(),
                    nat.ptr(offsets), nat.ptr(row_index), rows, M, x_int8.stride(0), N * K, N, K,
                    1 if offsets is None else w.shape[0], packed, nat.dtype_code(ws.dtype),
                    nat.dtype_code(b.dtype) if b is not None else 0, nat.dtype_code(out_dtype), act,
                    swiglu_alpha, swiglu_limit)
    with nat.on_device_of(x_int8):
        rc = nat.lib().ftm_w8a8_linear(ctypes.byref(c), nat.stream_of(x_int8))
    nat.check(rc, "ftm_w8a8_linear")
    return out


def w8a8_linear(
    x_int8: torch.Tensor,
    x_scale: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    *,
    bias: Optional[torch.Tensor] = None,
    activation: Optional[str] = None,
    swiglu_alpha: float = 1.702,
    swiglu_limit: float = 7.0,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """``(x_int8 @ weight.T) * x_scale[:, None] * weight_scale (+ bias)``, rounded once.

    ``x_int8 [M, K]`` and ``x_scale [M]`` as :func:`quantize_int8_token` gives them;
    ``weight`` int8 ``[N, K]`` or packed int32 ``[N, K/4]``, ``weight_scale [N]`` (or
    ``[N, 1]``).  With ``activation`` (as :class:`~ftmoe.layer.MoeLayer` names them) the
    weight's first N/2 rows are gate and the others up, and the result is
    ``act(gate) * up`` ``[M, N/2]``."""
    return _product(x_int8, x_scale, weight, weight_scale, offsets=None, row_index=None, bias=bias,
                    activation=activation, swiglu_alpha=swiglu_alpha, swiglu_limit=swiglu_limit, out_dtype=out_dtype)


def w8a8_grouped_linear(
    x_int8: torch.Tensor,
    x_scale: torch.Tensor,
    offsets: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    *,
    row_index: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    activation: Optional[str] = None,
    swiglu_alpha: float = 1.702,
    swiglu_limit: float = 7.0,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """:func:`w8a8_linear` of rows sorted by expert, each expert with a weight of its own.

    ``offsets`` int32 ``[E + 1]`` on the GPU, ascending: rows ``offsets[e]`` to
    ``offsets[e + 1]`` take ``weight[e]`` (``weight [E, N, K]`` or packed
    ``[E, N, K/4]``, ``weight_scale [E, N]``, ``bias [E, N]``); rows outside every
    expert's become zeros.  Without ``row_index`` the rows are those of ``x_int8``;
    with it (int32 ``[P]``, as ``TokenSort.token_of_row``) row r reads row
    ``row_index[r]`` of ``x_int8`` and ``x_scale``, and becomes zeros where that is no
    row.  E is at most 512."""
    for name, t in (("offsets", offsets), ("row_index", row_index)):
        if t is None:
            continue
        nat.require_gpu(t, name)
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
        if t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous and have one dimension, got {tuple(t.shape)}")
    if weight.dim() == 3 and offsets.shape[0] != weight.shape[0] + 1:
        raise ValueError(f"offsets must have {weight.shape[0] + 1} entries, got {offsets.shape[0]}")
    if not 1 <= offsets.shape[0] - 1 <= 512:
        raise ValueError(f"between 1 and 512 experts, got {offsets.shape[0] - 1}")
    return _product(x_int8, x_scale, weight, weight_scale, offsets=offsets, row_index=row_index, bias=bias,
                    activation=activation, swiglu_alpha=swiglu_alpha, swiglu_limit=swiglu_limit, out_dtype=out_dtype)


__all__ = ["quantize_int8_token", "w8a8_linear", "w8a8_grouped_linear"]
