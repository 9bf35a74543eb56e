"""Grouped GEMM of e4m3 rows and e4m3 expert weights with a scale for each block of 128 (csrc/fp8_gemm_sm100.cu).

Rows carry one fp32 scale for each 128 columns, weights one for each 128 x 128 block, of any positive value.  Half the bytes of the
bf16 experts in decode, twice the tensor rate in prefill.  Serving operators: they have no gradient, and with autograd on they refuse tensors that require one.
"""

from __future__ import annotations

import torch

from ..utils.build import load_extension as _ext
from .grouped_gemm import operator_status, refuse_gradients

BLOCK = 128
LARGEST = 448.0  # of e4m3
TINY = 1e-30     # smallest value that a block is scaled by


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16, fp16 or fp32 ``[rows, K]`` -> ``(q, scales)``: e4m3 ``[rows, K]`` and fp32 ``[rows, ceil(K / 128)]`` with ``q * scales = x``,
    ``scales = max(max |x|, 1e-30) / 448`` of each 128 columns."""
    refuse_gradients("quantize_rows", x)
    return _ext().quantize_rows(x)


@torch.no_grad()
def quantize_weights(w: torch.Tensor, *, swiglu: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``[E, N, K]`` or ``[N, K]`` weights -> e4m3 weights and a fp32 scale for each 128 x 128 block.  With ``swiglu`` (``N = 2 * I``: gate rows,
    then up rows) the halves have blocks of their own.  For loading a model: plain torch operations, one expert at a time;
    what it returns requires no gradient."""
    if w.dim() == 2:
        q, scales = quantize_weights(w[None], swiglu=swiglu)
        return q[0], scales[0]
    halves = 2 if swiglu else 1
    experts, rows, k = w.shape
    if rows % halves:
        raise ValueError("w must be [experts, 2 * I, K] with swiglu")
    part = rows // halves
    down, across = -(-part // BLOCK), -(-k // BLOCK)
    q = torch.empty(w.shape, dtype=torch.float8_e4m3fn, device=w.device)
    scales = torch.empty(experts, halves * down, across, dtype=torch.float32, device=w.device)
    for e in range(experts):
        for h in range(halves):
            mine = slice(h * part, (h + 1) * part)
            blocks = torch.nn.functional.pad(w[e, mine].float(), (0, across * BLOCK - k, 0, down * BLOCK - part)).view(down, BLOCK, across, BLOCK)
            largest = blocks.abs().amax((1, 3)).clamp_min(TINY)
            q[e, mine] = (blocks * LARGEST / largest[:, None, :, None]).reshape(down * BLOCK, across * BLOCK)[:part, :k].to(q.dtype)
            scales[e, h * down : (h + 1) * down] = largest / LARGEST
    return q, scales


def grouped_gemm_fp8(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, expert_offsets: torch.Tensor | None = None, *,
                     swiglu: bool = False, quantize: bool = False, row_scale: torch.Tensor | None = None, expert_counts: torch.Tensor | None = None,
                     max_expert_rows: int = 0):
    """``out[r] = (a[r] * a_scales[r]) @ (w[e(r)] * w_scales[e(r)]).T``, summed in FP32, to bf16 or (``quantize``) to ``(q, scales)`` as
    ``quantize_rows`` gives them, rounded from 32 bits.

    a: e4m3 ``[rows, K]`` with fp32 ``[rows, ceil(K / 128)]``; w: e4m3 ``[E, N, K]`` (``[E, 2 * I, K]``, gate rows then up rows, with ``swiglu``: the
    result is ``silu(gate) * up``) with fp32 ``[E, ceil(N / 128), ceil(K / 128)]`` (``2 * ceil(I / 128)``).  K, N and I are multiples of 16.
    ``w`` may be one matrix ``[N, K]``: a plain product, without ``expert_offsets``.
    expert_offsets: int64 ``[E + 1]``, not falling, from 0 to at most ``rows``, of any alignment; rows behind the last are not written.
    ``expert_counts`` (int64 ``[E]``): only so many rows of each range exist, the others are neither read nor written.
    ``row_scale`` (fp32 ``[rows]``, not with ``swiglu``) multiplies each output row before it is rounded.
    ``max_expert_rows`` (0 = unknown): no expert holds more rows.  The tile is chosen for so many rows where they are at most 32, else for the average of the
    ranges where that is less; it matters where ranges are padded, as behind a dispatch.  The result depends on it only in its rounding.
    """
    refuse_gradients("grouped_gemm_fp8", a, a_scales, w, w_scales, row_scale)
    if w.dim() == 2:
        w, w_scales = w[None], w_scales[None]
    out = _ext().grouped_gemm_fp8(a, a_scales, w, w_scales, expert_offsets, expert_counts, row_scale, bool(swiglu), bool(quantize),
                                  int(max_expert_rows), operator_status(a))
    return tuple(out) if quantize else out[0]
