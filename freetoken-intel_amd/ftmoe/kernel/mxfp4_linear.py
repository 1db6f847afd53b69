"""OCP MXFP4 weights (python/freetoken/kernel/triton/mxfp4_linear.py): 32 e2m1
values per block, 16 bytes, low nibble = even element, one e8m0 byte per block:
``value = LUT[nibble] * 2 ** (e8m0 - 127)`` computed on the GPU by ``ftm_dequant``."""
from __future__ import annotations

import ctypes
import math

import torch

from .. import _native as nat
from ..banks import FORMATS
from ..quant import quantize_mxfp4_blocks  # noqa: F401  (mxfp4_linear.py:79-111)


def dequantize_mxfp4_blocks(blocks: torch.Tensor, scales: torch.Tensor, *,
                            out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Dense ``[..., K]`` from ``blocks [..., n_blocks, 16]`` + ``scales [..., n_blocks]`` (mxfp4_linear.py:46-76)."""
    if blocks.dtype != torch.uint8:
        raise TypeError(f"MXFP4 blocks must be uint8, got {blocks.dtype}")
    if scales.dtype != torch.uint8:
        raise TypeError(f"MXFP4 scales must be uint8, got {scales.dtype}")
    if blocks.shape[-1] != 16:
        raise ValueError(f"MXFP4 block pack dimension must be 16 bytes, got {blocks.shape[-1]}")
    if blocks.shape[:-1] != scales.shape:
        raise ValueError(f"MXFP4 blocks/scales shape mismatch: {tuple(blocks.shape[:-1])} vs {tuple(scales.shape)}")
    nat.require_gpu(blocks, "weight")
    nat.require_gpu(scales, "weight")
    *lead, nb = scales.shape
    blocks, scales = blocks.contiguous(), scales.contiguous()
    out = torch.empty(*lead, nb * 32, dtype=out_dtype, device=blocks.device)
    p = nat.FtmProj(blocks.data_ptr(), scales.data_ptr(), None, None, 0, 0, 0, 0, FORMATS["mxfp4"], nat.DT_F32, nat.DT_BF16,
                    32, math.prod(lead), nb * 32, 1, 0)
    nat.launch("ftm_dequant", nat.lib().ftm_dequant, out, ctypes.byref(p), 0, out.data_ptr(), nat.dtype_code(out_dtype), 0)
    return out


def mxfp4_linear(x: torch.Tensor, weight_blocks: torch.Tensor, weight_scales: torch.Tensor, *,
                 bias: torch.Tensor | None = None) -> torch.Tensor:
    w = dequantize_mxfp4_blocks(weight_blocks, weight_scales, out_dtype=x.dtype)
    return torch.nn.functional.linear(x, w, bias)
