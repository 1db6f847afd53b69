"""MXFP4 activations x MXFP4 weights: the quantiser and the product of two
operands in blocks of 32 four-bit values (e2m1) with one power of two (e8m0)
each, dense or grouped by expert.  The reference has MXFP4 weights under wide
activations only (python/freetoken/kernel/triton/fused_mxfp4_linear.py); the
weights here are the same ``blocks`` and ``scales``.

gfx950: the scaled matrix instructions on 4-bit operands; a block's sum is exact,
blocks are added in fp32, bias and the gated activation are applied in fp32 in the
same kernel and rounded once.  For inference, like the other fused projections:
autograd does not see the calls."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .. import _native as nat
from ..layout import row_stride, rows_of
from .w8a8_linear import _dt, activation_code, bias_of

_QBLOCK = 32


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous, from a 16-byte border on."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def quantize_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [..., K]`` (fp32, fp16 or bf16; K a multiple of 32) -> (uint8 blocks
    ``[..., K/32, 16]``, uint8 e8m0 scales ``[..., K/32]``).  A block's scale is the least power of two 2^e with
    max |x| <= 6 * 2^e (the maximum taken as at least 1e-12); a value's code the nearest
    of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to |x| / 2^e, ties to the smaller.  A block with an
    infinity or NaN gets the scale 255 (NaN) and codes 0: its products are NaN, and so are its values.

    The rule of :func:`~ftmoe.quant.quantize_mxfp4_blocks`, and its bytes for every other block of bf16 or fp16; in
    fp32 that function finds e by a logarithm, which rounds to a whole number where the maximum is a few
    steps above 6 * 2^e (up to 33, where 2^e is far from 1): there it keeps e, this has e + 1."""
    nat.require_gpu(x, "x")
    dt = _dt(x.dtype, "x")
    if x.dim() == 0 or x.shape[-1] == 0 or x.shape[-1] % _QBLOCK != 0:
        raise ValueError(f"x must be [..., K] with K a multiple of {_QBLOCK}, got {tuple(x.shape)}")
    lead, K = x.shape[:-1], x.shape[-1]
    x2 = rows_of(x if x.dim() == 2 else x.reshape(-1, K))
    blocks = torch.empty(*lead, K // _QBLOCK, 16, dtype=torch.uint8, device=x.device)
    scales = torch.empty(*lead, K // _QBLOCK, dtype=torch.uint8, device=x.device)
    if x2.shape[0]:
        nat.launch("ftm_quant_mxfp4", nat.lib().ftm_quant_mxfp4, x2, x2.data_ptr(), dt, x2.shape[0], K,
                   row_stride(x2) * x2.element_size(), blocks.data_ptr(), scales.data_ptr())
    return blocks, scales


def mxfp4_of(blocks: torch.Tensor, scales: torch.Tensor, lead: int, name: str) -> tuple[torch.Tensor, torch.Tensor]:
    """(blocks, scales) as the kernels take them; ``lead`` dimensions before K/32."""
    if blocks.dtype != torch.uint8:
        raise TypeError(f"{name}_blocks must be uint8, got {blocks.dtype}")
    if scales.dtype != torch.uint8:
        raise TypeError(f"{name}_scales must be uint8, got {scales.dtype}")
    shape = blocks.shape
    if len(shape) != lead + 2 or shape[-1] != 16 or shape[-2] == 0:
        raise ValueError(f"{name}_blocks must be {['...'] * lead + ['K/32', 16]}, got {tuple(shape)}")
    if scales.shape != shape[:-1]:
        raise ValueError(f"{name}_scales must be {list(shape[:-1])}, got {tuple(scales.shape)}")
    if _QBLOCK * shape[-2] > nat.W4A4_MAX_K:
        raise ValueError(f"K={_QBLOCK * shape[-2]} exceeds {nat.W4A4_MAX_K}")
    return _aligned(blocks), scales.contiguous()


def _product(x, x_scales, weight_blocks, weight_scales, *, bias, out_dtype, offsets=None, row_index=None, activation=None,
             alpha=0.0, limit=0.0) -> torch.Tensor:
    """The call behind the products: x as codes with x_scales, or (x_scales None) wide x that the
    same call quantises."""
    nat.require_gpu(x, "x_blocks" if x_scales is not None else "x")
    nat.require_same_device(x, (("weight_blocks", weight_blocks), ("weight_scales", weight_scales),
                                ("x_scales", x_scales), ("bias", bias), ("offsets", offsets), ("row_index", row_index)))
    if x_scales is None:
        if x.dim() != 2 or x.shape[1] == 0 or x.shape[1] % _QBLOCK != 0:
            raise ValueError(f"x must be [M, K] with K a multiple of {_QBLOCK}, got {tuple(x.shape)}")
        x_dt = _dt(x.dtype, "x")
        M, K = x.shape
        x = rows_of(x)
    else:
        x, x_scales = mxfp4_of(x, x_scales, 1, "x")
        M, K = x.shape[0], _QBLOCK * x.shape[1]
    w, ws = mxfp4_of(weight_blocks, weight_scales, 1 if offsets is None else 2, "weight")
    if _QBLOCK * w.shape[-2] != K:
        raise ValueError(f"x's K={K} does not match weight_blocks' implied K={_QBLOCK * w.shape[-2]}")
    lead = w.shape[:-2]
    N = lead[-1]
    b, b_dt = bias_of(bias, lead, "bias")
    out_dt = _dt(out_dtype, "out_dtype")
    act = -1
    if activation is not None:
        act = activation_code(activation)
        if N % 2:
            raise ValueError(f"a gated activation needs an even number of weight rows (gate, then up), got {N}")
    rows = M if row_index is None else row_index.shape[0]
    out = torch.empty(rows, N // 2 if act >= 0 else N, dtype=out_dtype, device=x.device)
    if rows == 0 or N == 0:
        return out
    if M == 0:  # an index into no rows
        return out.zero_()
    nb = K // _QBLOCK
    if x_scales is None:  # codes, then the scales
        # held until the native call has enqueued its kernels: what is freed earlier another
        # thread may be given, and write, between the quantiser and the product
        scratch = torch.empty(17 * M * nb, dtype=torch.uint8, device=x.device)
        q, s = scratch.data_ptr(), scratch.data_ptr() + 16 * M * nb
    else:
        q, s = x.data_ptr(), x_scales.data_ptr()
    c = nat.FtmW4A4(q, s, w.data_ptr(), ws.data_ptr(), nat.ptr(b), out.data_ptr(), nat.ptr(offsets), nat.ptr(row_index),
                    rows, M, N * nb * 16, N * nb, N, K, 1 if offsets is None else lead[0], b_dt, out_dt, act, alpha, limit)
    if x_scales is None:
        nat.launch("ftm_w4a4_linear_dynamic", nat.lib().ftm_w4a4_linear_dynamic, x, x.data_ptr(), x_dt,
                   row_stride(x) * x.element_size(), ctypes.byref(c))
    else:
        nat.launch("ftm_w4a4_linear", nat.lib().ftm_w4a4_linear, x, ctypes.byref(c))
    return out


def w4a4_linear(
    x_blocks: torch.Tensor,
    x_scales: torch.Tensor,
    weight_blocks: torch.Tensor,
    weight_scales: torch.Tensor,
    *,
    bias: Optional[torch.Tensor] = None,
    activation: Optional[str] = None,
    swiglu_alpha: float = 1.702,
    swiglu_limit: float = 7.0,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """``deq(x) @ deq(weight).T (+ bias)``, fp32 sums, rounded once.

    ``x_blocks [M, K/32, 16]`` and ``x_scales [M, K/32]`` as :func:`quantize_mxfp4` gives
    them; ``weight_blocks [N, K/32, 16]``, ``weight_scales [N, K/32]``.  With ``activation``
    (as :class:`~ftmoe.layer.MoeLayer` names them) the weight's first N/2 rows are gate and
    the others up, and the result is ``act(gate) * up`` ``[M, N/2]``."""
    return _product(x_blocks, x_scales, weight_blocks, weight_scales, bias=bias, activation=activation,
                    alpha=swiglu_alpha, limit=swiglu_limit, out_dtype=out_dtype)


def w4a4_grouped_linear(
    x_blocks: torch.Tensor,
    x_scales: torch.Tensor,
    offsets: torch.Tensor,
    weight_blocks: torch.Tensor,
    weight_scales: torch.Tensor,
    *,
    row_index: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    activation: Optional[str] = None,
    swiglu_alpha: float = 1.702,
    swiglu_limit: float = 7.0,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """:func:`w4a4_linear` of rows sorted by expert, each expert with a weight of its own.

    ``offsets`` int32 ``[E + 1]`` on the GPU, ascending: rows ``offsets[e]`` to
    ``offsets[e + 1]`` take ``weight_blocks[e]`` (``weight_blocks [E, N, K/32, 16]``,
    ``weight_scales [E, N, K/32]``, ``bias [E, N]``); rows outside every expert's become
    zeros.  Without ``row_index`` the rows are those of ``x_blocks``; with it (int32
    ``[P]``, as ``TokenSort.token_of_row``) row r reads row ``row_index[r]``, and becomes
    zeros where that is no row.  E is at most 512."""
    for name, t in (("offsets", offsets), ("row_index", row_index)):
        if t is None:
            continue
        nat.require_gpu(t, name)
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
        if t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous and have one dimension, got {tuple(t.shape)}")
    E = offsets.shape[0] - 1
    if weight_blocks.dim() == 4 and weight_blocks.shape[0] != E:
        raise ValueError(f"offsets must have {weight_blocks.shape[0] + 1} entries, got {E + 1}")
    if not 1 <= E <= 512:
        raise ValueError(f"between 1 and 512 experts, got {E}")
    return _product(x_blocks, x_scales, weight_blocks, weight_scales, offsets=offsets, row_index=row_index, bias=bias,
                    activation=activation, alpha=swiglu_alpha, limit=swiglu_limit, out_dtype=out_dtype)


__all__ = ["quantize_mxfp4", "w4a4_linear", "w4a4_grouped_linear"]
