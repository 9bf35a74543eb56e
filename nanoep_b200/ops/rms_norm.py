"""Root-mean-square norm with the residual's addition and an output in 8 bits (csrc/rms_norm.cu).

The norm in front of an expert layer makes what the layer's dispatch moves and its products read: rows in 16 bits for the router
and a shared expert, e4m3 rows with a scale for each 128 columns for 8-bit experts, from one pass over the residual stream.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ..utils.build import load_extension as _ext
from .grouped_gemm import refuse_captured_gradients


class NormResult(NamedTuple):
    """``y`` ``[T, H]`` in the rows' type; ``q`` e4m3 ``[T, H]`` with ``scales`` fp32 ``[T, ceil(H / 128)]``; ``residual`` = x + residual in the rows'
    type (what was normalised, and what the next layer adds to); ``rstd`` fp32 ``[T]``.  ``None`` where not asked for."""

    y: torch.Tensor | None
    q: torch.Tensor | None
    scales: torch.Tensor | None
    residual: torch.Tensor | None
    rstd: torch.Tensor | None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6, quantize: bool = False,
             keep: bool = True, save: bool = False) -> NormResult:
    """``h = x + residual``; ``y = h * rsqrt(mean(h^2) + eps) * weight``.

    ``x`` and ``residual``: contiguous bf16, fp16 or fp32 ``[T, H]``; ``weight`` ``[H]`` of their type or fp32.  ``h`` is rounded to the rows' type before it
    is normalised, so that the norm of the returned ``residual`` is the same.  ``quantize``: also in e4m3, ``q * scales = y`` with
    ``scales = max |y| / 448`` of each 128 columns (at least 1e-30 / 448 in units of ``rstd``), rounded from 32 bits and not from ``y``.
    ``keep=False`` leaves ``y`` out; ``save`` returns ``rstd`` for ``rms_norm_grad``.  Differentiable in ``x``, ``residual`` and ``weight`` through
    ``y`` and ``residual``, once; the 8-bit form carries no gradient.
    """
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        if not keep:
            raise ValueError("gradients pass through y: keep=True")
        refuse_captured_gradients("rms_norm", "rms_norm_grad")
        return NormResult(*_ext().rms_norm_node(x, weight, residual, float(eps), bool(quantize), bool(save)))
    return NormResult(*_ext().rms_norm(x, weight, residual, float(eps), bool(quantize), bool(keep), bool(save)))


def rms_norm_grad(grad_y: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, *, grad_residual: torch.Tensor | None = None):
    """Gradients ``(grad_x, grad_weight)`` of ``rms_norm``; ``grad_x`` is that of ``residual`` as well.  ``h`` is what was normalised (the
    returned ``residual``, or ``x`` without one), ``grad_residual`` the gradient of the returned ``residual``.  Sums have one order on every run."""
    return _ext().rms_norm_grad(grad_y, h, weight, rstd, grad_residual)
