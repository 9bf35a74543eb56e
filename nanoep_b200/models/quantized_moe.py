"""Expert layer of one GPU with experts held in 8 bits, norm included.

    h = x + residual;  n = rms_norm(h) in e4m3
    y[t] = sum_k w[t,k] * W2[e_k] @ q( silu(W1g[e_k] @ n[t]) * (W1u[e_k] @ n[t]) )

The layer of ``moe_layer.ExpertParallelMoE`` without a group: no peer window and no wait of the host, so a step can be captured in a
CUDA graph.  Rows travel between its kernels in 8 bits with a scale for each 128 columns; down-projected rows in bf16.  It serves: the experts
have no gradient, so with autograd on (outside of ``torch.no_grad()``) nothing that comes into the layer may require one.
"""

from __future__ import annotations

import torch

from ..ops.fp8_gemm import grouped_gemm_fp8, quantize_rows, quantize_weights
from ..ops.grouped_gemm import refuse_gradients
from ..ops.rms_norm import rms_norm
from ..ops.token_order import plan_tokens, sort_tokens, unsort_tokens


class QuantizedMoE:
    """``w13`` e4m3 ``[E, 2 * I, H]`` (gate rows, then up rows) with ``w13_scales`` ``[E, 2 * ceil(I / 128), ceil(H / 128)]``, ``w2`` e4m3 ``[E, H, I]`` with
    ``w2_scales`` ``[E, ceil(H / 128), ceil(I / 128)]``.  ``norm_weight`` ``[H]``: the layer norms its input (and adds the residual) itself."""

    def __init__(self, w13: torch.Tensor, w13_scales: torch.Tensor, w2: torch.Tensor, w2_scales: torch.Tensor, *,
                 norm_weight: torch.Tensor | None = None, eps: float = 1e-6):
        if w13.dim() != 3 or w13.shape[1] % 32 or w13.shape[2] % 16:
            raise ValueError("w13 must be [experts, 2 * I, hidden] with I and hidden multiples of 16")
        if w2.shape != (w13.shape[0], w13.shape[2], w13.shape[1] // 2):
            raise ValueError("w2 must be [experts, hidden, I]")
        if w13.dtype != torch.float8_e4m3fn or w2.dtype != torch.float8_e4m3fn:
            raise ValueError("expert weights must be float8_e4m3fn (quantize() takes others)")
        self.w13, self.w13_scales, self.w2, self.w2_scales = w13, w13_scales, w2, w2_scales
        self.norm_weight, self.eps = norm_weight, eps
        self.num_experts = w13.shape[0]

    @classmethod
    def quantize(cls, w13: torch.Tensor, w2: torch.Tensor, **kwargs) -> "QuantizedMoE":
        """From weights in 16 or 32 bits."""
        return cls(*quantize_weights(w13, swiglu=True), *quantize_weights(w2), **kwargs)

    def forward(self, x: torch.Tensor, topk_idx: torch.Tensor | None = None, topk_weights: torch.Tensor | None = None, *,
                residual: torch.Tensor | None = None, router=None, bias: torch.Tensor | None = None):
        """``x`` ``[T, H]`` bf16, fp16 or fp32 (with a norm: ``norm_weight`` of that type or fp32); ``topk_idx`` int64 ``[T, K]`` (-1 = masked) and ``topk_weights`` fp32 ``[T, K]``, or ``router``, which gives both from the normed rows.
        Returns ``out`` bf16 ``[T, H]`` (plus ``bias`` bf16 ``[T, H]``, a shared expert's output), or ``(out, x + residual)`` where a ``residual`` is given."""
        refuse_gradients("QuantizedMoE", x, topk_weights, residual, bias, self.norm_weight, self.w13, self.w13_scales, self.w2, self.w2_scales)
        stream = None
        if self.norm_weight is not None:
            normed = rms_norm(x, self.norm_weight, residual=residual, eps=self.eps, quantize=True, keep=router is not None)
            rows, q, scales, stream = normed.y, normed.q, normed.scales, normed.residual
        elif residual is not None:
            raise ValueError("a residual is added by the layer's norm: norm_weight is needed")
        else:
            rows = x
            q, scales = quantize_rows(x)
        if router is not None:
            topk_idx, topk_weights = router(rows)
            refuse_gradients("QuantizedMoE", topk_weights)
        order = plan_tokens(topk_idx, self.num_experts)
        q, scales = sort_tokens(q, order, scales=scales)
        q, scales = grouped_gemm_fp8(q, scales, self.w13, self.w13_scales, order.expert_offsets, swiglu=True, quantize=True)
        y = grouped_gemm_fp8(q, scales, self.w2, self.w2_scales, order.expert_offsets)
        out = unsort_tokens(y, order, topk_weights, bias=bias)
        return out if stream is None else (out, stream)

    __call__ = forward
