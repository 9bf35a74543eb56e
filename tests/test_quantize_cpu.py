"""8-bit weights with a scale for each 128 x 128 block, and refusals that need no GPU."""

import pytest
import torch

from nanoep_b200.models.quantized_moe import QuantizedMoE
from nanoep_b200.ops.fp8_gemm import grouped_gemm_fp8, quantize_rows, quantize_weights
from nanoep_b200.ops.rms_norm import rms_norm
from nanoep_b200.ops.token_order import TokenOrder, plan_tokens, sort_tokens
from nanoep_b200.utils.build import load_extension


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


def _needs(t):
    return t.detach().clone().requires_grad_()


def test_operators_without_a_gradient_refuse_tensors_that_need_one():
    """Otherwise the result is a constant to autograd, and what is made of it a function of less than it is."""
    x = torch.ones(4, 128)
    (q, s), one = quantize_weights(torch.ones(128, 128)), torch.ones(4, 1)
    rows = torch.ones(4, 128).to(torch.float8_e4m3fn)
    for bad in (
        lambda: quantize_rows(_needs(x)),
        lambda: grouped_gemm_fp8(rows, _needs(one), q, s),
        lambda: grouped_gemm_fp8(rows, one, q, _needs(s)),
        lambda: grouped_gemm_fp8(rows, one, q, s, row_scale=_needs(one[:, 0])),
    ):
        with pytest.raises(ValueError, match="no gradient"):
            bad()
        with torch.no_grad(), pytest.raises((RuntimeError, ValueError), match="CUDA"):  # the next check
            bad()
    order = TokenOrder(*(torch.zeros(1, dtype=torch.int32) for _ in range(4)))
    with pytest.raises(ValueError, match="no gradient"):
        sort_tokens(rows, order, scales=_needs(one))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("which", ["x", "residual", "norm_weight", "topk_weights", "bias", "router"])
def test_the_layer_refuses_inputs_that_need_a_gradient(norm, which):
    if not norm and which in ("residual", "norm_weight"):
        pytest.skip("the norm's")
    weight = torch.ones(128) if norm else None
    layer = QuantizedMoE.quantize(torch.ones(2, 64, 128), torch.ones(2, 128, 32), norm_weight=_needs(weight) if which == "norm_weight" else weight)
    given = dict(x=torch.ones(4, 128), topk_idx=torch.zeros(4, 1, dtype=torch.int64), topk_weights=torch.ones(4, 1))
    if which in ("residual", "bias"):
        given[which] = torch.ones(4, 128)
    if which in given:
        given[which] = _needs(given[which])
    if which == "router":
        del given["topk_idx"], given["topk_weights"]
        given.update(x=_needs(given["x"]), router=lambda rows: pytest.fail("nothing runs before the refusal"))
    with pytest.raises(ValueError, match="QuantizedMoE has no gradient"):
        layer(**given)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):  # the next check: the operators'
        layer(**given)


def test_weights_in_8_bits_need_no_gradient():
    """Of a model's parameters: the layer takes what comes back."""
    q, s = quantize_weights(_needs(torch.randn(2, 160, 144)))
    assert not q.requires_grad and not s.requires_grad
    layer = QuantizedMoE.quantize(torch.nn.Parameter(torch.ones(2, 64, 128)), torch.nn.Parameter(torch.ones(2, 128, 32)))
    assert not any(t.requires_grad for t in (layer.w13, layer.w13_scales, layer.w2, layer.w2_scales))


@pytest.mark.parametrize("most", [1, 8, 16, 31, 33, 48, 64, 100])
@pytest.mark.parametrize("experts", [1, 4, 32, 256])
@pytest.mark.parametrize("swiglu", [False, True])
def test_a_hint_goes_for_padded_ranges(most, experts, swiglu):
    """Ranges of 128 rows in which no expert has more than ``most``: the kernel is that of ranges without padding."""
    def choice(rows, hint):
        return load_extension().fp8_gemm_choice(rows, experts, hint, 16, swiglu, 56, 148)

    assert choice(experts * 128, most) == choice(experts * most, most)
    assert choice(experts * 128, 128) == choice(experts * 128, 0) == choice(experts * 128, 5000)


def test_few_rows_in_padded_ranges_run_on_tiles_of_few_rows():
    choice = load_extension().fp8_gemm_choice
    assert choice(4096, 32, 0, 16, True, 56, 148)[0] == 128
    assert choice(4096, 32, 8, 16, True, 56, 148)[0] == choice(4096, 32, 32, 16, True, 56, 148)[0] == 32
    for swiglu in (False, True):
        assert choice(128, 1, 1, 16, swiglu, 56, 148) == choice(1, 1, 1, 16, swiglu, 56, 148)
