"""Norm with the residual's addition and the 8-bit output, against the formula in 64 bits.

Tolerances.  A rounding to type t is off by at most eps(t) / 2 relative.  In 32 bits: the sum of squares of H <= 40000 values is added in
chains of at most H / 512 + 21 (a thread's columns, the warp, the warps), under 2^-24 each, halved by the root; rsqrtf and the two
products add under 2^-21: together below 2^-17 for every H here.
"""

import pytest
import torch

from nanoep_b200.ops.fp8_gemm import quantize_rows
from nanoep_b200.ops.rms_norm import rms_norm, rms_norm_grad

pytestmark = pytest.mark.gpu
EPS32 = 2.0**-17
SMALLEST = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24, torch.float32: 2.0**-126}


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _reference(x, weight, residual, eps):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = h.double() * weight.double()
    rstd = (h.double().square().mean(-1, keepdim=True) + eps).rsqrt()
    return h, v, rstd


def _blocks(v):
    pad = -v.shape[1] % 128
    return torch.nn.functional.pad(v, (0, pad)).view(v.shape[0], -1, 128)


def _check_quantized(q, scales, v, rstd, exact):
    """q against v * 448 / max |v|; bit for bit where v is a product of two 16-bit values: the quotient in 32 bits is a tie only where it is one."""
    blocks = _blocks(v)
    most = blocks.abs().amax(-1).clamp_min(1e-30)
    want = (blocks * 448 / most[..., None]).view(v.shape[0], -1)[:, : v.shape[1]]
    torch.testing.assert_close(scales.double(), most * rstd / 448, rtol=EPS32, atol=0)
    if exact:
        assert torch.equal(q.float(), want.to(torch.float8_e4m3fn).float())
    else:
        # half a step of e4m3 (2^-4 relative, 2^-10 among the denormals) around a quotient that is off by 2^-22 at most
        assert bool(((q.double() - want).abs() <= want.abs() * (2.0**-4 + 2.0**-21) + 2.0**-10).all())


@pytest.mark.parametrize("tokens,hidden", [(1, 128), (1, 7168), (3, 8), (5, 1000), (2, 1), (7, 129), (33, 4096), (2, 8200), (2, 16392), (3, 40000), (700, 520)])
@pytest.mark.parametrize("dtype,wide", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False), (torch.float16, True), (torch.float32, False)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_forward(tokens, hidden, dtype, wide, with_residual):
    torch.manual_seed(tokens * hidden)
    x = torch.randn(tokens, hidden, device="cuda").to(dtype)
    residual = (torch.randn(tokens, hidden, device="cuda") * 3).to(dtype) if with_residual else None
    weight = (torch.randn(hidden, device="cuda") * 0.3 + 1).to(torch.float32 if wide else dtype)
    got = rms_norm(x, weight, residual=residual, eps=1e-5, quantize=True, save=True)
    h, v, rstd = _reference(x, weight, residual, 1e-5)
    if with_residual:
        assert torch.equal(got.residual, h)
    else:
        assert got.residual is None
    torch.testing.assert_close(got.rstd.double(), rstd[:, 0], rtol=EPS32, atol=0)
    torch.testing.assert_close(got.y.double(), v * rstd, rtol=_half_step(dtype) + 2 * EPS32, atol=SMALLEST[dtype])
    _check_quantized(got.q, got.scales, v, rstd, exact=dtype != torch.float32 and not wide)
    alone = rms_norm(x, weight, residual=residual, eps=1e-5)
    only = rms_norm(x, weight, residual=residual, eps=1e-5, quantize=True, keep=False)
    assert alone.q is None and only.y is None and torch.equal(alone.y, got.y)
    assert torch.equal(only.q.view(torch.uint8), got.q.view(torch.uint8)) and torch.equal(only.scales, got.scales)


@pytest.mark.parametrize("tokens,hidden", [(5000, 520), (1000, 7168), (700, 16384)])
@pytest.mark.parametrize("dtype,wide", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False), (torch.float32, False)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_several_rows_a_block(tokens, hidden, dtype, wide, with_residual):
    """More rows than twice the blocks of a launch: the next row's loads under the row before, sums by turns, in every width of a thread."""
    units = hidden // 8
    per = 1 if units <= 512 else 2 if units <= 1024 else 4
    threads = -(-(-(-units // per)) // 32) * 32
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert tokens > 2 * sms * max(1, min(16, (1536 if per == 1 else 1024) // threads)) and per == (1, 2, 4)[(520, 7168, 16384).index(hidden)]
    gen = torch.Generator(device="cuda").manual_seed(hidden)
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype) * torch.exp2(torch.randint(-3, 4, (tokens, 1), generator=gen, device="cuda")).to(dtype)
    residual = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype) if with_residual else None
    weight = (torch.randn(hidden, generator=gen, device="cuda") * 0.3 + 1).to(torch.float32 if wide else dtype)
    got = rms_norm(x, weight, residual=residual, eps=1e-5, quantize=True, save=True)
    for first in range(0, tokens, 1000):
        part = slice(first, first + 1000)
        h, v, rstd = _reference(x[part], weight, residual[part] if with_residual else None, 1e-5)
        assert not with_residual or torch.equal(got.residual[part], h)
        torch.testing.assert_close(got.rstd[part].double(), rstd[:, 0], rtol=EPS32, atol=0)
        torch.testing.assert_close(got.y[part].double(), v * rstd, rtol=_half_step(dtype) + 2 * EPS32, atol=SMALLEST[dtype])
        _check_quantized(got.q[part], got.scales[part], v, rstd, exact=False)


def test_gradients_of_both_inputs_are_tensors_of_their_own():
    """x and the residual have the same gradient; a step that changes one in place leaves the other."""
    x, r = (torch.randn(4, 64, device="cuda", requires_grad=True) for _ in range(2))
    got = rms_norm(x, torch.ones(64, device="cuda"), residual=r)
    g = torch.randn(4, 64, device="cuda")
    torch.autograd.backward((got.y, got.residual), (g, g))
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
    x.grad, r.grad = None, None
    rms_norm(x, torch.ones(64, device="cuda"), residual=r).residual.backward(g)
    x.grad.zero_()
    assert bool(r.grad.any()) and bool(g.any())


def test_rows_that_do_not_start_on_16_bytes():
    x = torch.randn(4, 256, device="cuda").to(torch.bfloat16)
    shifted = torch.empty(4 * 256 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(4, 256)
    shifted.copy_(x)
    weight = torch.randn(256, device="cuda").to(torch.bfloat16)
    a, b = (rms_norm(t, weight, quantize=True) for t in (x, shifted))
    # the two kernels add the squares in another order: y may round the other way, the 8-bit values do not depend on the sum
    torch.testing.assert_close(a.y.float(), b.y.float(), rtol=2 * _half_step(torch.bfloat16) + 2 * EPS32, atol=0)
    assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8))


def test_zero_rows_infinities_and_nan():
    x = torch.randn(5, 384, device="cuda").to(torch.bfloat16)
    x[0] = 0
    x[1, 7] = float("inf")
    x[2, 200] = float("nan")
    x[3, :128] = 0
    weight = torch.ones(384, device="cuda", dtype=torch.bfloat16)
    got = rms_norm(x, weight, quantize=True)
    assert torch.equal(got.y[0], torch.zeros_like(got.y[0])) and not got.q[0].float().any() and bool((got.scales[0] > 0).all())
    assert bool(got.y[2].isnan().all()) and bool(got.scales[2].isnan().all())
    assert bool(got.scales[1, 0].isnan()) and bool(got.y[1, 7].isnan()) and not got.y[1, 8:].any()  # rstd is 0
    assert not got.q[3, :128].float().any() and bool(got.q[3, 128:].float().abs().amax() == 448)
    assert bool(got.y[4].isfinite().all())


@pytest.mark.parametrize("rows,columns", [(1, 128), (1, 16), (3, 129), (5, 8), (257, 4096), (2, 1000), (1, 7)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_rows(rows, columns, dtype):
    torch.manual_seed(rows)
    x = (torch.randn(rows, columns, device="cuda") * torch.logspace(-4, 3, rows, device="cuda")[:, None]).to(dtype)
    x[0, 0] = 0
    q, scales = quantize_rows(x)
    _check_quantized(q, scales, x.double(), torch.ones(rows, 1, device="cuda", dtype=torch.float64), exact=dtype != torch.float32)


def _nearest_e4m3(q):
    """64-bit quotients of at most 448 to e4m3, rounded once (a conversion by torch goes through 32 bits, and rounds twice)."""
    step = torch.exp2(torch.frexp(q.abs().clamp_min(2.0**-6)).exponent.double() - 4)
    return torch.round(q / step) * step


def _next_to_ties(v, m):
    """Which quotients v * 448 / m are ties between two e4m3 values, or within 2^-21 of one."""
    q = v.double() * 448 / m.double()
    t = q / torch.exp2(torch.frexp(q.clamp_min(2.0**-6)).exponent.double() - 4)
    return (t - t.floor() - 0.5).abs() < 2.0**-21 * t


def test_ties_of_fp16_products():
    """Products of 22 bits whose quotient is a tie or lies next to one: in 64 bits a quotient differs from a tie by 2^-31 at least."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    a, b, c, d = torch.randint(1024, 2048, (4, 1 << 25), generator=gen, device="cuda")
    a, b, c, d = (torch.cat([torch.tensor(first, device="cuda"), t]) for first, t in zip(([1327, 1197], [1721, 2011], [1483, 441 * 4], [1597, 2011]), (a, b, c, d)))
    # the second pair of the list: its quotient is 76, between 72 and 80, with the larger value four times as large
    c = c * torch.where(torch.arange(len(c), device="cuda") % 2 == 1, 4, 1)
    v, m = a * b, c * d
    at = ((v <= m) & _next_to_ties(v, m)).nonzero().flatten()[:120]
    assert len(at) == 120 and at[:2].tolist() == [0, 1]
    for extra in (0, 1):  # the second width takes the kernel of any width
        x, weight = torch.zeros(2, 128 * 120 + extra, device="cuda"), torch.ones(128 * 120 + extra, device="cuda")
        first = torch.arange(120, device="cuda") * 128
        x[0, first], x[0, first + 1], weight[first], weight[first + 1] = a[at].float(), c[at].float(), b[at].float(), d[at].float()
        x[1] = -x[0]
        got = rms_norm(x.half(), weight.half(), quantize=True)
        want = _nearest_e4m3(v[at].double() * 448 / m[at].double())
        assert torch.equal(got.q[0, first].double(), want) and torch.equal(got.q[1, first].double(), -want)
        assert bool((got.q[0, first + 1].double() == 448).all())


def test_ties_of_32_bit_values():
    """24-bit values on both sides of every tie, and on it."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    blocks = 4096
    m = torch.randint(1 << 23, 1 << 24, (blocks,), generator=gen, device="cuda").double()
    m[::2] = torch.randint(1 << 17, 1 << 18, (blocks // 2,), generator=gen, device="cuda") * 56  # ties of these are exact: 448 = 8 * 56
    ties = torch.tensor([t * 2.0**e for e in range(-4, 4) for t in range(17, 33, 2)] + [t * 2.0**-10 for t in (1, 3, 5, 7, 9, 11, 13, 15)], device="cuda", dtype=torch.float64)
    on = (ties * m[:, None] / 448).float()
    x = torch.zeros(blocks, 256, device="cuda")
    x[:, :72], x[:, 128:200] = on, torch.nextafter(on, torch.zeros_like(on))
    x[:, 72], x[:, 73:127], x[:, 200] = m.float(), torch.nextafter(on, torch.full_like(on, 1e30))[:, :54], m.float()
    x *= torch.where(torch.rand(blocks, 256, generator=gen, device="cuda") < 0.5, -1, 1)
    for scale in (1.0, 2.0**100, 2.0**-120):
        q, _ = quantize_rows(x * scale)
        assert torch.equal(q.double(), _nearest_e4m3(x.double() * 448 / m[:, None]))


def _gradients(h, weight, rstd, gy, gh):
    """The formula's gradients in 64 bits, and the size of what is added up in each."""
    xhat, gw = h.double() * rstd, gy.double() * weight.double()
    mean, size = (gw * xhat).mean(-1, keepdim=True), (gw * xhat).abs().mean(-1, keepdim=True)
    dx = rstd * (gw - xhat * mean)
    scale = rstd * (gw.abs() + xhat.abs() * size)
    if gh is not None:
        dx, scale = dx + gh.double(), scale + gh.double().abs()
    return dx, scale, (gy.double() * xhat).sum(0), (gy.double() * xhat).abs().sum(0)


@pytest.mark.parametrize("tokens,hidden", [(1, 128), (3, 1000), (2, 129), (301, 4096), (900, 512), (5, 16392), (2, 7)])
@pytest.mark.parametrize("dtype,wide", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False), (torch.float32, False)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_gradients(tokens, hidden, dtype, wide, with_residual):
    torch.manual_seed(tokens + hidden)
    x = torch.randn(tokens, hidden, device="cuda").to(dtype).requires_grad_()
    residual = (torch.randn(tokens, hidden, device="cuda") * 3).to(dtype).requires_grad_() if with_residual else None
    weight = (torch.randn(hidden, device="cuda") * 0.3 + 1).to(torch.float32 if wide else dtype).requires_grad_()
    gy = torch.randn(tokens, hidden, device="cuda").to(dtype)
    gh = torch.randn(tokens, hidden, device="cuda").to(dtype) if with_residual else None
    got = rms_norm(x, weight, residual=residual, quantize=True)
    leaves = (x, weight, residual) if with_residual else (x, weight)
    grads = torch.autograd.grad((got.y, got.residual) if with_residual else got.y, leaves, (gy, gh) if with_residual else gy)
    with torch.no_grad():
        h, _, rstd = _reference(x, weight, residual, 1e-6)
        dx, size, dw, dw_size = _gradients(h, weight, rstd, gy, gh)
        # dx: 32-bit arithmetic on terms of `size`, one rounding; dw: chains of rows of a block, of blocks and of eight parts
        assert bool(((grads[0].double() - dx).abs() <= _half_step(dtype) * dx.abs() + 2 * EPS32 * size + SMALLEST[dtype]).all())
        chain = tokens // 148 + 300 / 8 + 12
        wt = weight.dtype
        assert bool(((grads[1].double() - dw).abs() <= _half_step(wt) * dw.abs() + (EPS32 + chain * 2.0**-24) * dw_size + SMALLEST[wt]).all())
        if with_residual:
            assert torch.equal(grads[2], grads[0])
        saved = rms_norm(x, weight, residual=residual, save=True)
        again = rms_norm_grad(gy, h, weight, saved.rstd, grad_residual=gh)
        assert torch.equal(again[0], grads[0]) and torch.equal(again[1], grads[1]), "the same sums on every run"


def test_gradients_against_differences():
    """Central differences of the operator itself.  With steps of 2^-6 the third-order term stays below 2^-12 / 6 of the derivative's
    size times a small factor; the forward's own rounding is 2^-17 of the loss's terms over 2^-5."""
    torch.manual_seed(1)
    x, r, w = torch.randn(3, 96, device="cuda"), torch.randn(3, 96, device="cuda"), torch.rand(96, device="cuda") + 0.5
    gy, gh = torch.randn(3, 96, device="cuda"), torch.randn(3, 96, device="cuda")

    def loss(x, r, w):
        got = rms_norm(x, w, residual=r)
        return (got.y.double() * gy).sum() + (got.residual.double() * gh).sum()

    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    got = rms_norm(leaves[0], leaves[2], residual=leaves[1])
    grads = torch.autograd.grad((got.y, got.residual), leaves, (gy, gh))
    for i, t in enumerate((x, r, w)):
        d = torch.randn_like(t)
        d /= d.norm() / 4
        step = 2.0**-6
        moved = [[u + s * step * d if j == i else u for j, u in enumerate((x, r, w))] for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        want = (grads[i].double() * d.double()).sum()
        size = (grads[i].double() * d.double()).abs().sum()
        noise = 2.0**-17 * (gy.abs().sum() * 3 + gh.abs().sum()) / (2 * step) / 16
        assert abs(float(slope - want)) <= float(size) * 2.0**-7 + float(noise)


def test_gradient_of_the_stream_alone_and_without_rows():
    x = torch.randn(2, 64, device="cuda", requires_grad=True)
    r = torch.randn(2, 64, device="cuda")
    w = torch.ones(64, device="cuda", requires_grad=True)
    g = torch.randn(2, 64, device="cuda")
    dx, dw = torch.autograd.grad(rms_norm(x, w, residual=r).residual, (x, w), g, allow_unused=True)
    assert torch.equal(dx, g) and dw is None
    empty = torch.empty(0, 64, device="cuda", requires_grad=True)
    got = rms_norm(empty, w, quantize=True)
    dx, dw = torch.autograd.grad(got.y, (empty, w), torch.empty(0, 64, device="cuda"))
    assert got.q.shape == (0, 64) and got.scales.shape == (0, 1) and dx.shape == (0, 64) and not dw.any()


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("save", [False, True])
@pytest.mark.parametrize("with_residual", [False, True])
def test_what_was_not_asked_for_is_none(grad, quantize, save, with_residual):
    x, r, w = torch.randn(2, 64, device="cuda"), torch.randn(2, 64, device="cuda"), torch.ones(64, device="cuda", requires_grad=grad)
    got = rms_norm(x, w, residual=r if with_residual else None, quantize=quantize, save=save)
    assert [t is not None for t in got] == [True, quantize, quantize, with_residual, save]
    assert got.y.requires_grad == grad and (got.rstd is None or not got.rstd.requires_grad)


def test_differentiable_once():
    x = torch.randn(2, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(rms_norm(x, w).y.sum(), x, create_graph=True)
    total = (rms_norm(x, w).y * 2).sum() + (x * x).sum()
    total.backward()
    assert x.grad.isfinite().all() and w.grad.isfinite().all()


def test_captured_forward_and_explicit_gradients():
    x, r, g = (torch.randn(40, 512, device="cuda").to(torch.bfloat16) for _ in range(3))
    w = torch.rand(512, device="cuda").to(torch.bfloat16)

    def step():
        got = rms_norm(x, w, residual=r, quantize=True, save=True)
        return (got.y, got.q.view(torch.uint8), got.scales, got.residual, *rms_norm_grad(g, got.residual, w, got.rstd, grad_residual=g))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
        with pytest.raises(RuntimeError, match="rms_norm_grad"):
            rms_norm(x.detach().requires_grad_(), w)
    for _ in range(2):
        for t in (x, r, g):
            t.normal_()
        graph.replay()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_a_batch_on_another_stream():
    """A long queue on one stream and the call on another: ordered by the caller, and the outputs belong to the call's stream."""
    stream = torch.cuda.Stream()
    x = torch.randn(64, 4096, device="cuda")
    w = torch.ones(4096, device="cuda")
    want = rms_norm(x, w, quantize=True)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [rms_norm(x, w, quantize=True) for _ in range(20)]
    torch.cuda.current_stream().wait_stream(stream)
    for g in got:
        assert torch.equal(g.y, want.y) and torch.equal(g.scales, want.scales) and torch.equal(g.q.view(torch.uint8), want.q.view(torch.uint8))


def test_largest_values_of_the_type():
    """h * weight near the largest 32-bit value: neither the quotient nor the scale's product overflows where the result does not."""
    x = torch.full((1, 256), 2.0**126, device="cuda")
    x[0, 1::2] = 2.0**120
    q, scales = quantize_rows(x)
    assert torch.equal(q.float()[0, :2], torch.tensor([448.0, 7.0], device="cuda"))
    torch.testing.assert_close(q.double() * scales.double().repeat_interleave(128, 1), x.double(), rtol=2.0**-20, atol=0)


def test_refusals():
    x = torch.randn(2, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    for bad in (
        lambda: rms_norm(x.cpu(), w),
        lambda: rms_norm(x.t(), w),
        lambda: rms_norm(x.double(), w),
        lambda: rms_norm(x, w[:32]),
        lambda: rms_norm(x, w.to(torch.bfloat16)),
        lambda: rms_norm(x, w, residual=x.half()),
        lambda: rms_norm(x, w, residual=x[:1]),
        lambda: rms_norm(x, w, eps=-1.0),
        lambda: rms_norm(x, w, keep=False),
        lambda: rms_norm(x[0], w),
        lambda: rms_norm_grad(x, x, w, torch.ones(3, device="cuda")),
        lambda: quantize_rows(x.to(torch.int32)),
    ):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        rms_norm(x.requires_grad_(), w, quantize=True, keep=False)
