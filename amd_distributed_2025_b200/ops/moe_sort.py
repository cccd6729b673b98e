"""Tokens sorted by expert, and the weighted way back, for the experts that live on one GPU.

``MoEAllToAll`` delivers rows to a slab of ``max_recv`` rows for every expert.  Where all experts are local there are
only ``T * k`` rows: here they lie packed, expert by expert, in the order in which ``ops.fp8_gemm.fp8_grouped_gemm`` (or
a library's grouped product) takes them:

    sorted = sort_tokens(x, indices, num_experts)          # rows [T k, H], order (offsets, row_of)
    y = experts(sorted.rows, sorted.order.offsets)         # expert e: rows offsets[e] .. offsets[e + 1]
    out = unsort_tokens(y, sorted.order, weights)          # [T, H]

Inside an expert rows are in (token, k) order, as in the dispatch layout.  An entry whose id is not in
``[0, num_experts)`` (-1: an expert of another rank, or none) has no row and adds nothing; the rows behind the last
expert's are zero, in gradients too.  A token may name an expert twice and has two rows then.  Sums are fp32, over k
upwards, rounded once; nothing depends on an order of atomics.

Both are differentiable (fp16, bf16, fp32) in reverse mode; forward-mode tangents are refused.  The gradients can be had
without autograd too: ``sort_tokens_backward`` and ``unsort_tokens_backward``.  All of it may be captured into a CUDA graph;
a forward pass that is captured while an eager graph of the same leaves is alive is refused (their gradients are added up on
the eager graph's stream, for which a captured backward pass cannot wait).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _ext


_tuple = tuple.__new__  # (what the classes below do in Python on every call takes as long as a short kernel's launch)


class ExpertOrder(NamedTuple):
    """Where the rows of the entries lie."""

    offsets: torch.Tensor  # int32 [num_experts + 1]: expert e has rows offsets[e] .. offsets[e + 1]
    row_of: torch.Tensor  # int32 [T, k]: the row of each entry, or -1


class SortedTokens(NamedTuple):
    """What ``sort_tokens`` returns."""

    rows: torch.Tensor  # [T k, H] in x's type
    scale: Optional[torch.Tensor]  # float32 [T k, scales of a row], where scales were given
    order: ExpertOrder


def sort_tokens(
    x: torch.Tensor, indices: torch.Tensor, num_experts: int, *, scale: Optional[torch.Tensor] = None
) -> SortedTokens:
    """Copies row ``t`` of ``x [T, H]`` (fp16, bf16, fp32 or float8_e4m3fn) to a row for each of its experts
    ``indices [T, k]`` (int32 or int64, k <= 32, num_experts <= 8192), packed expert by expert.

    ``scale [T, S]`` (fp32) goes the same way: the block scales of e4m3 rows.  It has no gradient, and neither has ``x`` beside
    it: what wants one is refused."""
    ext = _ext.load()
    got = ext.sort_tokens(x, indices, num_experts, scale)
    if got is None:  # x wants a gradient
        if scale is not None or x.element_size() == 1:
            raise ValueError("e4m3 rows and rows with scales have no gradient: call sort_tokens under torch.no_grad()")
        _refuse_foreign_leaves(ext, x)
        rows, offsets, row_of = _Sort.apply(x, indices, num_experts)
        return SortedTokens(rows, None, ExpertOrder(offsets, row_of))
    rows, rows_scale, offsets, row_of = got
    return _tuple(SortedTokens, (rows, rows_scale, _tuple(ExpertOrder, (offsets, row_of))))


def unsort_tokens(rows: torch.Tensor, order: ExpertOrder, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * rows[row_of[t, j]]`` (weights of one where there are none), in the rows' type.

    ``rows [T k, H]`` in fp16, bf16 or fp32; ``weights [T, k]`` in a floating type."""
    ext = _ext.load()
    out = ext.unsort_tokens(rows, order.row_of, weights)
    if out is not None:
        return out
    if weights is not None and weights.dtype != torch.float32:
        if not weights.dtype.is_floating_point:
            raise ValueError(f"weights must be of a floating type, not {weights.dtype}")
        weights = weights.to(torch.float32)
        out = ext.unsort_tokens(rows, order.row_of, weights)
        if out is not None:  # nothing wants a gradient
            return out
    _refuse_foreign_leaves(ext, rows, weights)
    return _Unsort.apply(rows, order.offsets, order.row_of, weights)


def sort_tokens_backward(grad_rows: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """Gradient of ``x`` from that of ``sort_tokens(x, ...).rows``: each token's rows added up."""
    with torch.no_grad():
        return _ext.load().unsort_tokens(grad_rows, order.row_of, None)


def unsort_tokens_backward(
    grad: torch.Tensor, rows: torch.Tensor, order: ExpertOrder, weights: Optional[torch.Tensor] = None
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of ``rows`` and of ``weights`` (fp32; None without weights) from that of ``unsort_tokens(...)``."""
    if weights is not None and weights.dtype != torch.float32:
        weights = weights.detach().to(torch.float32)
    return _ext.load().unsort_tokens_backward(grad, rows, order.offsets, order.row_of, weights, True, True)


def _refuse_foreign_leaves(ext, *tensors: Optional[torch.Tensor]) -> None:
    on_gpu = [t for t in tensors if t is not None and t.is_cuda]
    if not on_gpu or not torch.cuda.is_current_stream_capturing():
        return
    for t in on_gpu:
        if ext.adds_up_elsewhere(t):
            raise RuntimeError("a backward pass cannot be captured while an eager graph of the same leaves is alive: "
                               "drop that graph (its outputs and losses) before the capture")


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, indices, num_experts):
        rows, _, offsets, row_of = _ext.load().sort_tokens(x, indices, num_experts, None)
        ctx.save_for_backward(row_of)
        ctx.mark_non_differentiable(offsets, row_of)
        ctx.set_materialize_grads(False)
        return rows, offsets, row_of

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_rows, *_):
        (row_of,) = ctx.saved_tensors
        grad_x = None if grad_rows is None else _ext.load().unsort_tokens(grad_rows, row_of, None)
        return grad_x, None, None


class _Unsort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, offsets, row_of, weights):
        ctx.save_for_backward(rows if ctx.needs_input_grad[3] else None, offsets, row_of, weights)
        return _ext.load().unsort_tokens(rows, row_of, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, offsets, row_of, weights = ctx.saved_tensors
        grad_rows, grad_weights = _ext.load().unsort_tokens_backward(
            grad, rows, offsets, row_of, weights, ctx.needs_input_grad[0], ctx.needs_input_grad[3])
        return grad_rows, None, None, grad_weights
