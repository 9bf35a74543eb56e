"""A batch sorted by expert and back on one GPU (csrc/token_order.cu): the local counterpart of dispatch and combine.

No peer window, no host wait for counts and a fixed row order: forward calls can be captured in a CUDA graph, and rows, outputs
and gate weights are differentiable (once).  ``slot`` is the row of one choice (token ``t``, choice ``k``); the rows of an expert are
ordered by (t, k).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ..utils.build import load_extension as _ext
from .grouped_gemm import operator_status, refuse_captured_gradients


class TokenOrder(NamedTuple):
    """``slots`` int32 ``[T, K]`` row of each choice (-1 = masked); ``slot_map`` int32 ``[C]`` choice ``t * K + k`` of each row (-1 = none);
    ``expert_counts`` int64 ``[E]``; ``expert_offsets`` int64 ``[E + 1]``, multiples of the alignment.  ``C`` (``capacity``) holds any
    routing of the batch: rows behind ``expert_offsets[E]`` belong to nobody."""

    slots: torch.Tensor
    slot_map: torch.Tensor
    expert_counts: torch.Tensor
    expert_offsets: torch.Tensor

    @property
    def capacity(self) -> int:
        return self.slot_map.shape[0]


def plan_tokens(topk_idx: torch.Tensor, num_experts: int, *, alignment: int = 1) -> TokenOrder:
    """Order of the choices ``topk_idx`` (int64 ``[T, K]``, expert ids or -1) by expert.

    Capacity is ``T * K + min(E, T * K) * (alignment - 1)``, rounded up to a multiple of ``alignment``.  An id outside ``[-1, E)`` is
    treated as masked and reported by ``grouped_gemm.check_status()``.
    """
    return TokenOrder(*_ext().plan_tokens(topk_idx, int(num_experts), int(alignment), operator_status(topk_idx)))


def sort_tokens(x: torch.Tensor, order: TokenOrder, *, scales: torch.Tensor | None = None, zero_padding: bool = False):
    """``rows[order.slots[t, k]] = x[t]``: bf16, fp16, fp32 or e4m3 ``[T, H]`` to ``[C, H]``.

    ``scales`` (fp32 ``[T, blocks]``, of 8-bit rows) travels along, and ``(rows, row_scales)`` is returned.  With ``zero_padding`` every row
    without a choice is zero, otherwise it is not written.  Differentiable in ``x`` (without ``scales``).
    """
    if torch.is_grad_enabled() and (x.requires_grad or (scales is not None and scales.requires_grad)):
        if scales is not None:
            raise ValueError("rows that travel with scales have no gradient")
        refuse_captured_gradients("sort_tokens", "sort_tokens_grad")
        return _ext().sort_tokens_node(x, order.slots, order.slot_map, bool(zero_padding))
    rows, row_scales = _ext().sort_tokens(x, order.slots, order.slot_map, scales, bool(zero_padding))
    return rows if scales is None else (rows, row_scales)


def unsort_tokens(y: torch.Tensor, order: TokenOrder, weights: torch.Tensor | None = None, *, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = bias[t] + sum_k weights[t, k] * y[order.slots[t, k]]``, summed in FP32 in ascending ``k`` and rounded once.

    ``y`` bf16, fp16 or fp32 ``[C, H]`` (rows without a choice are not read), ``weights`` fp32 ``[T, K]`` (ones without; those of masked
    choices may be anything), ``bias`` ``[T, H]`` of ``y``'s type.  Differentiable in all three.
    """
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, weights, bias)):
        refuse_captured_gradients("unsort_tokens", "unsort_tokens_grad")
        return _ext().unsort_tokens_node(y, order.slots, order.slot_map, weights, bias)
    return _ext().unsort_tokens(y, order.slots, order.slot_map, weights, bias)


def sort_tokens_grad(grad_rows: torch.Tensor, order: TokenOrder) -> torch.Tensor:
    """Gradient of ``sort_tokens`` in ``x``: the sum of a token's rows.  Rows without a choice are not read."""
    return _ext().unsort_tokens(grad_rows, order.slots, order.slot_map, None, None)


def unsort_tokens_grad(grad_out: torch.Tensor, y: torch.Tensor, order: TokenOrder, weights: torch.Tensor | None = None):
    """Gradients of ``unsort_tokens`` in ``y`` (zero in rows without a choice) and in ``weights`` (0 for masked choices; ``None`` without)."""
    return _ext().unsort_tokens_grad(grad_out, y, order.slots, order.slot_map, weights)
