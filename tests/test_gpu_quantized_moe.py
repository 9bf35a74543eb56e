"""The layer with experts in 8 bits: norm, order, products and back as they are used together.

Tolerance: held in 8 bits between its steps, a value is off by 2^-4 at most, the root of the mean square of a rounding within its step by
about 2^-4 / sqrt(3) = 0.036 at the coarse end of a binade.  The reference makes the same roundings from 64-bit sums; where a value lies next to a border
the layer's 32-bit sum may fall on the other side, an error of one step of one value in thousands.  2-norm of the difference below 0.02 of
the result leaves room for the bf16 roundings (2^-8 each) and for those; a missing or doubled row shows as a multiple of it."""

from datetime import timedelta

import pytest
import torch
import torch.distributed as dist

from nanoep_b200 import CudaBuffer, EPConfig
from nanoep_b200.models.quantized_moe import QuantizedMoE
from nanoep_b200.ops import grouped_gemm as gg
from nanoep_b200.ops.fp8_gemm import grouped_gemm_fp8, quantize_rows
from nanoep_b200.ops.rms_norm import rms_norm

pytestmark = pytest.mark.gpu


def _blockwise(v):
    """64-bit values held in e4m3 with a scale for each 128 columns."""
    n = v.shape[1]
    blocks = torch.nn.functional.pad(v, (0, -n % 128)).view(len(v), -1, 128)
    most = blocks.abs().amax(-1, keepdim=True).clamp_min(1e-30)
    return ((blocks * 448 / most).to(torch.float8_e4m3fn).double() * (most / 448)).view(len(v), -1)[:, :n]


def _full(w, scales, halves):
    E, n, k = w.shape
    s = scales.double().view(E, halves, -1, scales.shape[-1]).repeat_interleave(128, 2)[:, :, : n // halves].repeat_interleave(128, 3)[..., :k]
    return w.double() * s.reshape(E, n, k)


def _reference(layer, x, idx, gate, residual):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = h.double() * layer.norm_weight.double() if layer.norm_weight is not None else h.double()
    n = _blockwise(v)
    if layer.norm_weight is not None:
        n = n * (h.double().square().mean(-1, keepdim=True) + layer.eps).rsqrt()
    w13, w2 = _full(layer.w13, layer.w13_scales, 2), _full(layer.w2, layer.w2_scales, 1)
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for e in range(layer.num_experts):
        t, k = (idx == e).nonzero(as_tuple=True)
        if len(t):
            g, u = (n[t] @ w13[e].T).chunk(2, 1)
            y = (_blockwise(g * torch.sigmoid(g) * u) @ w2[e].T).to(torch.bfloat16).double()
            out.index_add_(0, t, y * gate[t, k].double()[:, None])
    return out, h


def _layer(experts, hidden, inner, norm=True):
    gen = torch.Generator(device="cuda").manual_seed(hidden)
    w13 = torch.randn(experts, 2 * inner, hidden, generator=gen, device="cuda") * hidden**-0.5
    w2 = torch.randn(experts, hidden, inner, generator=gen, device="cuda") * inner**-0.5
    weight = (torch.rand(hidden, generator=gen, device="cuda") + 0.5).to(torch.bfloat16) if norm else None
    return QuantizedMoE.quantize(w13.to(torch.bfloat16), w2.to(torch.bfloat16), norm_weight=weight)


def _batch(tokens, hidden, experts, topk, seed=0, masked=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").to(torch.bfloat16)
    gate, idx = torch.rand(tokens, experts, generator=gen, device="cuda").topk(topk, dim=-1)
    if masked:
        idx = idx.masked_fill(torch.rand(tokens, topk, generator=gen, device="cuda") < 0.2, -1)
    return x, idx, gate / gate.sum(-1, keepdim=True)


def _near(got, want):
    assert bool(got.isfinite().all())
    assert float((got.double() - want).norm()) <= 0.02 * float(want.norm())


@pytest.mark.parametrize("tokens,hidden,inner,experts,topk", [(1, 256, 128, 4, 2), (33, 512, 256, 8, 4), (200, 1040, 400, 3, 2), (7, 2048, 512, 64, 6), (600, 768, 384, 2, 2)])
@pytest.mark.parametrize("norm", [True, False])
def test_layer(tokens, hidden, inner, experts, topk, norm):
    layer = _layer(experts, hidden, inner, norm)
    x, idx, gate = _batch(tokens, hidden, experts, topk)
    out = layer(x, idx, gate)
    want, _ = _reference(layer, x, idx, gate, None)
    _near(out, want)
    bias = torch.randn(tokens, hidden, device="cuda").to(torch.bfloat16)
    _near(layer(x, idx, gate, bias=bias), want + bias.double())
    if norm:
        residual = torch.randn(tokens, hidden, device="cuda").to(torch.bfloat16)
        out, stream = layer(x, idx, gate, residual=residual)
        want, h = _reference(layer, x, idx, gate, residual)
        _near(out, want)
        assert torch.equal(stream, h)
    gg.check_status()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("norm", [True, False])
def test_rows_of_other_types(dtype, norm):
    """Rows in fp16 or fp32: the result stays bf16, and so does what is added to it."""
    layer = _layer(8, 512, 256, norm)
    if norm:
        layer.norm_weight = layer.norm_weight.to(dtype)
    x, idx, gate = _batch(70, 512, 8, 2)
    x, bias = x.to(dtype), torch.randn(70, 512, device="cuda").to(torch.bfloat16)
    want, _ = _reference(layer, x, idx, gate, None)
    out = layer(x, idx, gate, bias=bias)
    assert out.dtype == torch.bfloat16
    _near(out, want + bias.double())
    if norm:
        residual = torch.randn(70, 512, device="cuda").to(dtype)
        out, stream = layer(x, idx, gate, residual=residual)
        want, h = _reference(layer, x, idx, gate, residual)
        _near(out, want)
        assert stream.dtype == dtype and torch.equal(stream, h)
    with pytest.raises(RuntimeError, match="bias"):
        layer(x, idx, gate, bias=bias.to(dtype))


def test_between_dispatch_and_combine(monkeypatch):
    """The 8-bit products on a dispatch's rows: aligned ranges, counts that leave padding rows out, gate weights in the product, and a combine behind them."""
    monkeypatch.setenv("LOCAL_RANK", "0")
    monkeypatch.setenv("LOCAL_WORLD_SIZE", "1")
    layer = _layer(8, 512, 256, norm=False)
    x, idx, gate = _batch(300, 512, 8, 4)
    own = not dist.is_initialized()
    if own:
        dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1, timeout=timedelta(seconds=60))
    try:
        with CudaBuffer(dist.group.WORLD, EPConfig(8, 4, 512, 300)) as buf:
            got = buf.dispatch(x, topk_idx=idx, weights=gate, do_expand=True, alignment=128)
            layout = got.handle.layout
            ranges = dict(expert_counts=layout.expert_counts, max_expert_rows=layout.recv_count)
            q, scales = grouped_gemm_fp8(*quantize_rows(got.x), layer.w13, layer.w13_scales, layout.expert_offsets, swiglu=True, quantize=True, **ranges)
            y = grouped_gemm_fp8(q, scales, layer.w2, layer.w2_scales, layout.expert_offsets, row_scale=got.topk_weights, **ranges)
            out = buf.combine(y, got.handle).x
            torch.cuda.synchronize()
            buf.check_status()
            gg.check_status()
    finally:
        if own:
            dist.destroy_process_group()
    _near(out, _reference(layer, x, idx, gate, None)[0])


def test_router_sees_the_normed_rows():
    layer = _layer(8, 512, 256)
    x, idx, gate = _batch(40, 512, 8, 2, masked=False)
    seen = []
    out = layer(x, router=lambda rows: (seen.append(rows), (idx, gate))[1])
    assert torch.equal(seen[0], rms_norm(x, layer.norm_weight, eps=layer.eps).y)
    assert torch.equal(out, layer(x, idx, gate))


def test_parameters_are_served_without_autograd():
    """With autograd on, a router with parameters is refused like any input that needs a gradient; without, the layer gives what it gives for plain tensors."""
    layer = _layer(8, 512, 256)
    x, idx, gate = _batch(40, 512, 8, 2, masked=False)
    want = layer(x, idx, gate)
    scale = torch.nn.Parameter(torch.ones((), device="cuda"))
    with pytest.raises(ValueError, match="no gradient"):
        layer(x, router=lambda rows: (idx, gate * scale))
    layer.norm_weight = torch.nn.Parameter(layer.norm_weight)
    with pytest.raises(ValueError, match="no gradient"):
        layer(x, idx, gate)
    for off in (torch.no_grad(), torch.inference_mode()):
        with off:
            assert torch.equal(layer(x, router=lambda rows: (idx, gate * scale)), want)


def test_every_choice_masked():
    layer = _layer(4, 256, 128)
    x = torch.randn(5, 256, device="cuda").to(torch.bfloat16)
    out = layer(x, torch.full((5, 2), -1, device="cuda"), torch.full((5, 2), float("nan"), device="cuda"))
    assert not out.any()


def test_no_tokens():
    layer = _layer(4, 256, 128)
    out, stream = layer(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16), torch.empty(0, 2, dtype=torch.int64, device="cuda"), torch.empty(0, 2, device="cuda"),
                        residual=torch.empty(0, 256, device="cuda", dtype=torch.bfloat16))
    assert out.shape == stream.shape == (0, 256)


def test_two_layers_at_once():
    """Two layers on two streams share no state."""
    layers = [_layer(8, 512, 256), _layer(4, 1024, 128)]
    batches = [_batch(200, h, e, 2, s) for s, (h, e) in enumerate(((512, 8), (1024, 4)))]
    want = [layer(*batch) for layer, batch in zip(layers, batches)]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for layer, batch, stream in zip(layers, batches, streams):
            with torch.cuda.stream(stream):
                got.append(layer(*batch))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, want[i % 2])


def test_captured_step():
    layer = _layer(8, 512, 256)
    x, idx, gate = _batch(64, 512, 8, 4)
    residual = torch.randn_like(x)
    layer(x, idx, gate, residual=residual)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer(x, idx, gate, residual=residual)
    for seed in (1, 2):
        for mine, new in zip((x, idx, gate), _batch(64, 512, 8, 4, seed)):
            mine.copy_(new)
        graph.replay()
        again = layer(x, idx, gate, residual=residual)
        assert torch.equal(held[0], again[0]) and torch.equal(held[1], again[1])


def test_refusals():
    layer = _layer(4, 256, 128)
    with pytest.raises(ValueError):
        QuantizedMoE(layer.w13, layer.w13_scales, layer.w2[:, :128], layer.w2_scales)
    with pytest.raises(ValueError):
        QuantizedMoE(layer.w13.float(), layer.w13_scales, layer.w2, layer.w2_scales)
    with pytest.raises(ValueError):
        bare = QuantizedMoE(layer.w13, layer.w13_scales, layer.w2, layer.w2_scales)
        x, idx, gate = _batch(4, 256, 4, 2)
        bare(x, idx, gate, residual=x)
