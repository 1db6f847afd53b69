"""(token, expert) pairs sorted by expert, tokens copied into that order, and
rows back in token order with their router weights -- with gradients (reverse
mode), so a trained router or trained experts can stand between the two.

The grouping that the layer kernels do inside
(python/freetoken/kernel/triton/fused_moe.py:106-161), as operators: a stable
counting sort on the GPU, no atomics, no host synchronisation, the sums in a
fixed order (repeated calls give identical bits)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.function import once_differentiable

from .. import _native as nat
from ..layout import row_stride, rows_of

ID_DTYPES = {torch.int32: nat.ID_I32, torch.int64: nat.ID_I64}


@dataclass(frozen=True)
class TokenSort:
    """The order of ``T k`` pairs (pair ``p = t k + j``), all int32 on the GPU.

    Rows ``offsets[e]`` to ``offsets[e + 1]`` are expert e's pairs in order of p; the
    pairs without an expert follow from ``offsets[E]`` on.  ``row_of_pair [T, k]`` and
    ``pair_of_row [T k]`` are inverse to each other and hold the complement (``~row``,
    ``~pair``, so a negative number) for a pair without an expert; ``token_of_row`` is
    the pair's token, -1 without an expert."""

    num_experts: int
    offsets: torch.Tensor
    row_of_pair: torch.Tensor
    pair_of_row: torch.Tensor
    token_of_row: torch.Tensor


def sort_tokens(topk_ids: torch.Tensor, num_experts: int) -> TokenSort:
    """Sort the pairs of ``topk_ids [T, k]`` (int32 or int64) by expert, stably.  An id
    outside ``[0, num_experts)`` is a pair without an expert; ``num_experts`` <= 512."""
    nat.require_gpu(topk_ids, "topk_ids")
    if topk_ids.dtype not in ID_DTYPES:
        raise TypeError(f"topk_ids must be int32 or int64, got {topk_ids.dtype}")
    if topk_ids.dim() != 2 or topk_ids.shape[1] == 0:
        raise ValueError(f"topk_ids must be [T, k] with k > 0, got {tuple(topk_ids.shape)}")
    E = int(num_experts)
    if not 1 <= E <= 512:
        raise ValueError(f"between 1 and 512 experts, got {E}")
    ids = topk_ids.contiguous()
    T, k = ids.shape
    if T * k >= 2**31 - 1:
        raise ValueError(f"{T} x {k} pairs exceed 32 bits")
    L, dev = nat.lib(), ids.device
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    row_of_pair = torch.empty((T, k), dtype=torch.int32, device=dev)
    pair_of_row = torch.empty(T * k, dtype=torch.int32, device=dev)
    token_of_row = torch.empty(T * k, dtype=torch.int32, device=dev)
    need = L.ftm_sort_workspace_bytes(T, k, E)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    nat.launch("ftm_sort_tokens", L.ftm_sort_tokens, ids, ids.data_ptr(), ID_DTYPES[ids.dtype], T, k, E,
               offsets.data_ptr(), row_of_pair.data_ptr(), pair_of_row.data_ptr(), token_of_row.data_ptr(),
               nat.ptr(ws), need)
    return TokenSort(E, offsets, row_of_pair, pair_of_row, token_of_row)


def _check_sort(sort: TokenSort, t: torch.Tensor, name: str) -> None:
    nat.require_gpu(t, name)
    r = sort.row_of_pair
    if r.dtype != torch.int32 or r.dim() != 2 or not r.is_contiguous():
        raise ValueError("the sort's row_of_pair must be a contiguous int32 [T, k]")
    if r.device != t.device:
        raise ValueError(f"the sort is on {r.device}, {name} on {t.device}")


def _gather(x: torch.Tensor, sort: TokenSort) -> torch.Tensor:
    T, k = sort.row_of_pair.shape
    x = rows_of(x)
    H, size = x.shape[1], x.element_size()
    rows = torch.empty((T * k, H), dtype=x.dtype, device=x.device)
    if rows.numel() == 0:
        return rows
    nat.launch("ftm_gather_tokens", nat.lib().ftm_gather_tokens, x, x.data_ptr(), row_stride(x) * size, size, H,
               sort.row_of_pair.data_ptr(), T, k, rows.data_ptr())
    return rows


def _combine(rows: torch.Tensor, w: Optional[torch.Tensor], sort: TokenSort, out_dtype: torch.dtype) -> torch.Tensor:
    T, k = sort.row_of_pair.shape
    rows = rows_of(rows)
    H = rows.shape[1]
    out = torch.empty((T, H), dtype=out_dtype, device=rows.device)
    if out.numel() == 0:
        return out
    w = w.contiguous() if w is not None else None
    nat.launch("ftm_combine_tokens", nat.lib().ftm_combine_tokens, rows, rows.data_ptr(), nat.dtype_code(rows.dtype),
               row_stride(rows) * rows.element_size(), nat.ptr(w), nat.dtype_code(w.dtype) if w is not None else 0,
               sort.row_of_pair.data_ptr(), T, k, H, out.data_ptr(), nat.dtype_code(out_dtype))
    return out


def _refuse_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """The kernels know nothing of forward mode: a tangent would be dropped."""
    for t in tensors:
        if t is not None and fwAD.unpack_dual(t).tangent is not None:
            raise NotImplementedError("gather_tokens and combine_tokens have no forward-mode derivative")


def _first_only(backward):
    """``backward``, refusing a second derivative, in forward mode too; the wrapper that
    refuses one in reverse mode costs more than a small backward itself, so it is passed
    only where one may follow."""
    once = once_differentiable(backward)

    def run(ctx, g):
        _refuse_tangents(g)
        return once(ctx, g) if torch.is_grad_enabled() else backward(ctx, g)

    return run


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, sort):
        ctx.sort = sort
        ctx.save_for_backward(sort.row_of_pair)  # a later write to it is found
        return _gather(x, sort)

    @staticmethod
    @_first_only
    def backward(ctx, g):
        ctx.saved_tensors
        return _combine(g, None, ctx.sort, g.dtype), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, w, sort, out_dtype):
        ctx.sort = sort
        ctx.save_for_backward(rows, w, sort.row_of_pair)
        return _combine(rows, w, sort, out_dtype)

    @staticmethod
    @_first_only
    def backward(ctx, g):
        rows, w, row_of_pair = ctx.saved_tensors
        T, k = row_of_pair.shape
        want_rows, want_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        g, rows, wc = rows_of(g), rows_of(rows), w.contiguous()
        H = rows.shape[1]
        grad_rows = torch.empty((T * k, H), dtype=rows.dtype, device=rows.device) if want_rows else None
        grad_w = torch.empty((T, k), dtype=w.dtype, device=w.device) if want_w else None
        if T == 0 or H == 0:
            return grad_rows, None if grad_w is None else grad_w.zero_(), None, None
        nat.launch("ftm_combine_tokens_grad", nat.lib().ftm_combine_tokens_grad, rows, g.data_ptr(),
                   nat.dtype_code(g.dtype), row_stride(g) * g.element_size(), rows.data_ptr(),
                   nat.dtype_code(rows.dtype), row_stride(rows) * rows.element_size(), wc.data_ptr(),
                   nat.dtype_code(w.dtype), row_of_pair.data_ptr(), T, k, H, nat.ptr(grad_rows), nat.ptr(grad_w))
        return grad_rows, grad_w, None, None


def _recorded(*inputs: Optional[torch.Tensor]) -> bool:
    """Whether autograd has to see the call."""
    _refuse_tangents(*inputs)
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs)


def gather_tokens(x: torch.Tensor, sort: TokenSort) -> torch.Tensor:
    """``x [T, H]`` -> ``[T k, H]``: row r is token ``sort.token_of_row[r]``, zeros where
    that is -1.  Any dtype of 1, 2 or 4 bytes; differentiable in x (fp32, fp16, bf16; in
    reverse mode, once): a token's gradient is the sum of its rows', in fp32, rounded once."""
    _check_sort(sort, x, "x")
    if x.dim() != 2 or x.shape[0] != sort.row_of_pair.shape[0]:
        raise ValueError(f"x must be [{sort.row_of_pair.shape[0]}, H], got {tuple(x.shape)}")
    if x.element_size() not in (1, 2, 4):
        raise TypeError(f"x must have elements of 1, 2 or 4 bytes, got {x.dtype}")
    if _recorded(x):
        nat.dtype_code(x.dtype)
        return _Gather.apply(x, sort)
    return _gather(x, sort)


def combine_tokens(rows: torch.Tensor, topk_w: Optional[torch.Tensor], sort: TokenSort, *,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``rows [T k, H]`` (sorted order) -> ``[T, H]``: the sum over j of ``topk_w[t, j]``
    times the row of pair (t, j), pairs without an expert left out (their rows are not
    read); fp32 sums in order of j, rounded once.  ``rows`` and ``topk_w [T, k]`` in
    fp32, fp16 or bf16 (``topk_w`` None: ones), ``out_dtype`` the rows' (the default) or,
    from fp32 rows, any of the three.  Differentiable in both (in reverse mode, once): rows
    of no expert get zero gradients, and so do their weights."""
    _check_sort(sort, rows, "rows")
    T, k = sort.row_of_pair.shape
    nat.dtype_code(rows.dtype)
    out_dtype = out_dtype if out_dtype is not None else rows.dtype
    nat.dtype_code(out_dtype)
    if out_dtype != rows.dtype and rows.dtype != torch.float32:
        raise TypeError(f"rows of {rows.dtype} are summed to {rows.dtype}, not {out_dtype}")
    if rows.dim() != 2 or rows.shape[0] != T * k:
        raise ValueError(f"rows must be [{T * k}, H], got {tuple(rows.shape)}")
    if topk_w is not None:
        nat.dtype_code(topk_w.dtype)
        nat.require_same_device(rows, (("topk_w", topk_w),))
        if tuple(topk_w.shape) != (T, k):
            raise ValueError(f"topk_w must be [{T}, {k}], got {tuple(topk_w.shape)}")
    if _recorded(rows, topk_w):
        if topk_w is None:
            topk_w = torch.ones((T, k), dtype=torch.float32, device=rows.device)
        return _Combine.apply(rows, topk_w, sort, out_dtype)
    return _combine(rows, topk_w, sort, out_dtype)


__all__ = ["TokenSort", "sort_tokens", "gather_tokens", "combine_tokens"]
