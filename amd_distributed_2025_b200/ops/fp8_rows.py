"""Rows for the fp8 GEMMs: e4m3 values with one fp32 scale for each row and 128 columns.

``fp8_gemm`` and ``fp8_grouped_gemm`` take their left operand as ``(a [M, K], a_scale [M, ceil(K/128)])``.  These
operators leave it in one pass over what comes before a product:

* ``rms_norm_fp8``: ``h = x + residual``, ``y = h * rsqrt(mean(h^2) + eps) * weight``;
* ``silu_mul_fp8``: ``y = g / (1 + exp(-g)) * u`` for ``x = [g | u]``, between the two products of a gated expert.

Of a block of 128 columns (the last one of a row may be shorter) ``scale = max(max|y|, 1e-30) / 448`` and
``q = e4m3(y / scale)``, rounded to nearest even; a block with a NaN in it is NaN in every place, its scale among them, and
beside an infinity what is finite is zero.
All of it is fp32 between the loads and the one rounding of each output (csrc/fp8_rows.cu); a row whose squares add up to
more than fp32 holds is normed to zeros.

Inputs are CUDA matrices in fp16, bf16 or fp32 (all of a call of one type; the weight may be fp32 beside the others),
with any distance between rows; rows that are not contiguous are copied first.  The operators have no gradient, in
neither mode, and refuse inputs that want one.  They launch on the current stream of the inputs' device.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _ext


class NormedRows(NamedTuple):
    """What ``rms_norm_fp8`` returns."""

    q: torch.Tensor  # float8_e4m3fn [rows, columns]
    scale: torch.Tensor  # float32 [rows, ceil(columns / 128)]
    total: Optional[torch.Tensor]  # x + residual in x's type; None without a residual
    normed: Optional[torch.Tensor]  # y in x's type, where it was asked for


def rms_norm_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    residual: Optional[torch.Tensor] = None,
    total_out: Optional[torch.Tensor] = None,
    normed: bool = False,
) -> NormedRows:
    """Root-mean-square norm of each row of ``x + residual``, quantised.

    ``total`` is the sum, rounded to x's type (the norm is taken of the unrounded one); ``total_out`` may be ``residual``
    or ``x`` itself, which is then overwritten, or a matrix that overlaps neither.  ``normed=True`` gives the normed
    rows in x's type as well (a router reads them).  At most 32768 columns."""
    return NormedRows(*_ext.load().rms_norm_fp8(x, weight, eps, residual, total_out, normed))


def silu_mul_fp8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q [rows, columns], scale [rows, ceil(columns/128)])`` of ``silu(x[:, :columns]) * x[:, columns:]``."""
    return _ext.load().silu_mul_fp8(x)
