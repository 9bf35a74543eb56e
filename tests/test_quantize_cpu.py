"""8-bit weights with a scale for each 128 x 128 block, and refusals that need no GPU."""

import pytest
import torch

from nanoep_b200.ops.fp8_gemm import grouped_gemm_fp8, quantize_rows, quantize_weights
from nanoep_b200.ops.rms_norm import rms_norm
from nanoep_b200.ops.token_order import plan_tokens


@pytest.mark.parametrize("shape,swiglu", [((2, 256, 128), False), ((1, 16, 16), False), ((3, 272, 144), False), ((2, 2 * 144, 272), True), ((130, 260), False)])
def test_weights(shape, swiglu):
    torch.manual_seed(0)
    w = torch.randn(shape)
    w.view(-1)[:5] = 0
    q, scales = quantize_weights(w, swiglu=swiglu)
    halves = 2 if swiglu else 1
    n, k = shape[-2:]
    full = scales.double().view(-1, halves, scales.shape[-2] // halves, scales.shape[-1])
    full = full.repeat_interleave(128, 2)[:, :, : n // halves].repeat_interleave(128, 3)[..., :k].reshape(shape)
    # half a step of e4m3: 2^-4 relative, 2^-10 of the scale among the denormals; the quotient and the scale in 32 bits add 2^-21
    assert q.shape == w.shape and bool(((q.double() * full - w.double()).abs() <= w.double().abs() * (2.0**-4 + 2.0**-21) + 2.0**-10 * full).all())
    assert float(q.float().abs().max()) == 448


def test_a_block_of_zeros_has_a_scale():
    q, scales = quantize_weights(torch.zeros(1, 128, 128))
    assert not q.float().any() and bool((scales > 0).all())


def test_refusals():
    with pytest.raises(ValueError):
        quantize_weights(torch.zeros(1, 7, 16), swiglu=True)
    x = torch.zeros(2, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        rms_norm(x, torch.ones(128))
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        plan_tokens(torch.zeros(2, 1, dtype=torch.int64), 4)
    q, s = quantize_weights(torch.ones(128, 128))
    with pytest.raises(ValueError, match="CUDA"):
        grouped_gemm_fp8(q, s, q, s)
