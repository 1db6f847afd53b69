"""Int8 activations x int8 weights: the per-token quantiser and the integer
product with one scale per token and one per output channel, dense or grouped
by expert.  The reference has INT8 weights under wide activations only
(python/freetoken/kernel/triton/fused_int8_linear.py); the weights here are the
same codes and scales, either plain int8 ``[N, K]``
(:func:`~ftmoe.quant.quantize_int8_channel`) or the checkpoint's packed int32
``[N, K/4]`` (offset-binary bytes, one scale a row).

gfx950: int32 sums on the int8 matrix cores, exact for K up to 131071, so a
result does not depend on the batch it is computed in; scales, bias and the
gated activation are applied in fp32 in the same kernel and rounded once.  For
inference, like the other fused projections: autograd does not see the calls."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .. import _native as nat
from ..layer import ACTIVATIONS
from ..layout import row_stride, rows_of

_DT = {torch.float32: nat.DT_F32, torch.float16: nat.DT_F16, torch.bfloat16: nat.DT_BF16}


def _dt(dtype, name: str) -> int:
    code = _DT.get(dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {dtype}")
    return code


def quantize_int8_token(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [..., K]`` (fp32, fp16 or bf16) -> (int8 codes ``[..., K]``, fp32 scales
    ``[...]``): scale = max |x| / 127 of the row (the maximum at least 1e-12; times the
    fp32 nearest 1 / 127, as torch divides by a number on the GPU), code = the whole
    number nearest x / scale, ties to even.  A row with an infinity or
    NaN gets the scale NaN and codes 0: its products are NaN, no other row's are."""
    nat.require_gpu(x, "x")
    dt = _dt(x.dtype, "x")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., K] with K > 0, got {tuple(x.shape)}")
    lead, K = x.shape[:-1], x.shape[-1]
    x2 = rows_of(x if x.dim() == 2 else x.reshape(-1, K))
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(lead, dtype=torch.float32, device=x.device)
    if x2.shape[0]:
        nat.launch("ftm_quant_int8", nat.lib().ftm_quant_int8, x2, x2.data_ptr(), dt, x2.shape[0], K,
                   row_stride(x2) * x2.element_size(), q.data_ptr(), K, scale.data_ptr())
    return q, scale


def weight_of(weight: torch.Tensor, K: int, dim: int, name: str = "weight") -> tuple[torch.Tensor, int]:
    """(contiguous weight, whether it is packed) for activations of K channels."""
    if weight.dtype == torch.int8:
        packed, k = 0, weight.shape[-1] if weight.dim() else 0
    elif weight.dtype == torch.int32:
        packed, k = 1, 4 * weight.shape[-1] if weight.dim() else 0
    else:
        raise TypeError(f"{name} must be int8 or packed int32, got {weight.dtype}")
    if weight.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, got shape {tuple(weight.shape)}")
    if k != K:
        raise ValueError(f"x's K={K} does not match the {name}'s K={k}")
    if K > nat.W8A8_MAX_K:
        raise ValueError(f"K={K} exceeds {nat.W8A8_MAX_K}: int32 sums of int8 products could overflow")
    return weight.contiguous(), packed


def scale_of(t: torch.Tensor, shape, name: str) -> tuple[torch.Tensor, int]:
    """(contiguous scales of ``shape`` -- or with a last 1, one group a row --, their dtype code)."""
    code = _dt(t.dtype, name)
    if t.shape != shape and t.shape != (*shape, 1):
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    return t.contiguous(), code


def bias_of(t: Optional[torch.Tensor], shape, name: str) -> tuple[Optional[torch.Tensor], int]:
    if t is None:
        return None, 0
    code = _dt(t.dtype, name)
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    return t.contiguous(), code


def activation_code(activation: str) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"unsupported MoE activation: {activation!r}")
    return ACTIVATIONS[activation]


def _product(x, x_scale, weight, weight_scale, *, bias, out_dtype, offsets=None, row_index=None, activation=None,
             alpha=0.0, limit=0.0) -> torch.Tensor:
    """The call behind the products: x int8 with x_scale, or (x_scale None) wide x that the
    same call quantises."""
    nat.require_gpu(x, "x_int8" if x_scale is not None else "x")
    nat.require_same_device(x, (("weight", weight), ("weight_scale", weight_scale), ("x_scale", x_scale),
                                ("bias", bias), ("offsets", offsets), ("row_index", row_index)))
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"x must be [M, K] with K > 0, got {tuple(x.shape)}")
    M, K = x.shape
    if x_scale is None:
        x_dt = _dt(x.dtype, "x")
    else:
        if x.dtype != torch.int8:
            raise TypeError(f"x_int8 must be int8, got {x.dtype}")
        if x_scale.dtype != torch.float32:
            raise TypeError(f"x_scale must be float32, got {x_scale.dtype}")
        if x_scale.shape != (M,) and x_scale.shape != (M, 1):
            raise ValueError(f"x_scale must be [{M}], got {tuple(x_scale.shape)}")
        x_scale = x_scale.contiguous()
    w, packed = weight_of(weight, K, 2 if offsets is None else 3)
    lead = w.shape[:-1]
    N = lead[-1]
    ws, ws_dt = scale_of(weight_scale, lead, "weight_scale")
    b, b_dt = bias_of(bias, lead, "bias")
    out_dt = _dt(out_dtype, "out_dtype")
    act = -1
    if activation is not None:
        act = activation_code(activation)
        if N % 2:
            raise ValueError(f"a gated activation needs an even number of weight rows (gate, then up), got {N}")
    x = rows_of(x)
    rows = M if row_index is None else row_index.shape[0]
    out = torch.empty((rows, N // 2 if act >= 0 else N), dtype=out_dtype, device=x.device)
    if out.numel() == 0:
        return out
    if M == 0:  # an index into no rows
        return out.zero_()
    if x_scale is None:  # codes, then the scales on a 4-byte border
        at = (M * K + 3) // 4 * 4
        # held until the native call has enqueued its kernels: what is freed earlier another
        # thread may be given, and write, between the quantiser and the product
        scratch = torch.empty(at + 4 * M, dtype=torch.uint8, device=x.device)
        q, s, stride = scratch.data_ptr(), scratch.data_ptr() + at, K
    else:
        x = x if row_stride(x) >= K else x.contiguous()  # rows over one another
        q, s, stride = x.data_ptr(), x_scale.data_ptr(), row_stride(x)
    c = nat.FtmW8A8(q, s, w.data_ptr(), ws.data_ptr(), None if b is None else b.data_ptr(), out.data_ptr(),
                    None if offsets is None else offsets.data_ptr(), None if row_index is None else row_index.data_ptr(),
                    rows, M, stride, N * K, N, K, 1 if offsets is None else lead[0], packed, ws_dt, b_dt, out_dt, act,
                    alpha, limit)
    if x_scale is None:
        nat.launch("ftm_w8a8_linear_dynamic", nat.lib().ftm_w8a8_linear_dynamic, x, x.data_ptr(), x_dt,
                   row_stride(x) * x.element_size(), ctypes.byref(c))
    else:
        nat.launch("ftm_w8a8_linear", nat.lib().ftm_w8a8_linear, x, ctypes.byref(c))
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
    return _product(x_int8, x_scale, weight, weight_scale, bias=bias, activation=activation, alpha=swiglu_alpha,
                    limit=swiglu_limit, out_dtype=out_dtype)


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
    E = offsets.shape[0] - 1
    if weight.dim() == 3 and weight.shape[0] != E:
        raise ValueError(f"offsets must have {weight.shape[0] + 1} entries, got {E + 1}")
    if not 1 <= E <= 512:
        raise ValueError(f"between 1 and 512 experts, got {E}")
    return _product(x_int8, x_scale, weight, weight_scale, offsets=offsets, row_index=row_index, bias=bias,
                    activation=activation, alpha=swiglu_alpha, limit=swiglu_limit, out_dtype=out_dtype)


__all__ = ["quantize_int8_token", "w8a8_linear", "w8a8_grouped_linear"]
