"""Tensors of more than 2^31 elements: rows at the far end are those of the same rows alone."""

import pytest
import torch

from nanoep_b200.ops import grouped_gemm as gg
from nanoep_b200.ops.fp8_gemm import quantize_rows, quantize_weights
from nanoep_b200.ops.rms_norm import rms_norm, rms_norm_grad
from nanoep_b200.ops.token_order import TokenOrder, sort_tokens, unsort_tokens, unsort_tokens_grad

pytestmark = pytest.mark.gpu
ROWS, HIDDEN = 300_007, 7168
FAR = slice(ROWS - 301, ROWS)


@pytest.fixture()
def rows():
    assert ROWS * HIDDEN > 2**31
    x = torch.empty(ROWS, HIDDEN, dtype=torch.bfloat16, device="cuda")
    x.view(-1)[: 1 << 24].normal_()
    for first in range(1 << 24, x.numel(), 1 << 24):  # copies of other rows: only the far ones count
        part = x.view(-1)[first : first + (1 << 24)]
        part.copy_(x.view(-1)[: part.numel()])
    x[FAR].normal_()
    yield x
    del x
    torch.cuda.empty_cache()


def test_norm_and_its_gradient(rows):
    weight = torch.rand(HIDDEN, device="cuda").to(torch.bfloat16)
    got, part = (rms_norm(t, weight, quantize=True, save=True) for t in (rows, rows[FAR].contiguous()))
    for name in ("y", "q", "scales", "rstd"):
        assert torch.equal(getattr(got, name)[FAR].view(torch.uint8), getattr(part, name).view(torch.uint8)), name
    dx, _ = rms_norm_grad(rows, rows, weight, got.rstd)
    assert torch.equal(dx[FAR], rms_norm_grad(rows[FAR].contiguous(), rows[FAR].contiguous(), weight, part.rstd)[0])
    del dx
    q, scales = quantize_rows(rows)
    part = quantize_rows(rows[FAR].contiguous())
    assert torch.equal(q[FAR].view(torch.uint8), part[0].view(torch.uint8)) and torch.equal(scales[FAR], part[1])


def test_order(rows):
    """300 tokens whose rows lie at the far end of the order."""
    tokens = 300
    slots = torch.arange(ROWS - tokens, ROWS, device="cuda", dtype=torch.int32).view(tokens, 1)
    slot_map = torch.full((ROWS,), -1, dtype=torch.int32, device="cuda")
    slot_map[-tokens:] = torch.arange(tokens, device="cuda", dtype=torch.int32)
    order = TokenOrder(slots, slot_map, torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"))
    x, weights = torch.randn(tokens, HIDDEN, device="cuda").to(torch.bfloat16), torch.rand(tokens, 1, device="cuda")
    out = sort_tokens(x, order, zero_padding=True)
    assert torch.equal(out[-tokens:], x) and not out[-2 * tokens : -tokens].any() and not out[:tokens].any()
    del out
    assert torch.equal(unsort_tokens(rows, order, weights), (rows[-tokens:].float() * weights).to(torch.bfloat16))
    dy, _ = unsort_tokens_grad(x, rows, order, weights)
    assert torch.equal(dy[-tokens:], (x.float() * weights).to(torch.bfloat16)) and not dy[-2 * tokens : -tokens].any()


@pytest.mark.parametrize("tile", [64, 128])
def test_product(tile):
    """Operand rows, then output rows, that end behind 2^31 bytes and elements."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    for k, n in ((HIDDEN, 128), (16, HIDDEN)):
        a = torch.empty(ROWS, k, dtype=torch.float8_e4m3fn, device="cuda")
        a.view(torch.uint8).fill_(0x38)
        a[FAR] = torch.randn(301, k, generator=gen, device="cuda").to(a.dtype)
        scales = torch.rand(ROWS, -(-k // 128), generator=gen, device="cuda")
        w, w_scales = quantize_weights(torch.randn(n, k, generator=gen, device="cuda"))

        def product(a, scales):
            offsets = torch.tensor([0, len(a)], device="cuda")
            return gg._ext().grouped_gemm_fp8(a, scales, w[None], w_scales[None], offsets, None, None, False, False, 0, gg.status_tensor(a.device), tile, 1, 0)[0]

        out = product(a, scales)
        gg.check_status()
        torch.testing.assert_close(out[FAR].float(), product(a[FAR].contiguous(), scales[FAR].contiguous()).float(), rtol=0, atol=0)
        del out, a
    torch.cuda.empty_cache()
