"""Tensor layouts that the kernels take."""
from __future__ import annotations

import torch


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """``t [n, H]`` with neighbouring elements of a row side by side (rows may lie apart)."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def row_stride(t: torch.Tensor) -> int:
    """Elements between the rows of ``t`` (a single row may carry any stride)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]
