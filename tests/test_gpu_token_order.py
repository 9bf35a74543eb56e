"""A batch sorted by expert and back, against a plain implementation; sums against 64 bits.

Tolerances: a sum of n products in 32 bits is off by at most (n + 1) * 2^-24 of the sum of their sizes (fused multiply-adds), and a
rounding to type t by eps(t) / 2 of the result."""

import pytest
import torch

from nanoep_b200.ops import grouped_gemm as gg
from nanoep_b200.ops.token_order import plan_tokens, sort_tokens, sort_tokens_grad, unsort_tokens, unsort_tokens_grad

pytestmark = pytest.mark.gpu
SMALLEST = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24, torch.float32: 2.0**-126}


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _order(idx, experts, alignment):
    choice = idx.flatten().tolist()
    counts = [sum(c == e for c in choice) for e in range(experts)] if experts * len(choice) < 10**6 else torch.bincount(
        torch.tensor([c for c in choice if c >= 0], dtype=torch.int64), minlength=experts).tolist()
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + -(-c // alignment) * alignment)
    capacity = -(-(len(choice) + min(experts, len(choice)) * (alignment - 1)) // alignment) * alignment
    assert offsets[-1] <= capacity
    at, slots, slot_map = offsets[:-1].copy(), [], [-1] * capacity
    for i, e in enumerate(choice):
        slots.append(at[e] if e >= 0 else -1)
        if e >= 0:
            slot_map[at[e]] = i
            at[e] += 1
    return torch.tensor(slots, dtype=torch.int32).view(idx.shape), torch.tensor(slot_map, dtype=torch.int32), torch.tensor(counts), torch.tensor(offsets)


def _routing(tokens, experts, topk, kind, seed=0):
    gen = torch.Generator().manual_seed(seed + tokens)
    if kind == "same":  # the same index in every choice
        return torch.full((tokens, topk), experts - 1, dtype=torch.int64)
    if kind == "masked":
        return torch.full((tokens, topk), -1, dtype=torch.int64)
    idx = torch.randint(-1 if kind == "some masked" else 0, experts, (tokens, topk), generator=gen)
    if kind == "skewed":
        idx = (torch.rand(tokens, topk, generator=gen) ** 4 * experts).long()
    return idx


@pytest.mark.parametrize("tokens,experts,topk", [(0, 4, 2), (1, 1, 1), (1, 256, 8), (3, 5, 32), (37, 64, 6), (129, 1024, 8), (1025, 60, 1), (4096, 256, 8), (20011, 33, 3)])
@pytest.mark.parametrize("alignment", [1, 16, 128])
@pytest.mark.parametrize("kind", ["uniform", "some masked", "skewed", "same", "masked"])
def test_plan(tokens, experts, topk, alignment, kind):
    idx = _routing(tokens, experts, topk, kind)
    got = plan_tokens(idx.cuda(), experts, alignment=alignment)
    for name, mine, want in zip(got._fields, got, _order(idx, experts, alignment)):
        assert torch.equal(mine.cpu(), want.to(mine.dtype)), name
    gg.check_status()


@pytest.mark.parametrize("dtype,hidden", [(torch.bfloat16, 256), (torch.bfloat16, 7168), (torch.bfloat16, 2), (torch.bfloat16, 129), (torch.float16, 1000),
                                          (torch.float32, 515), (torch.float8_e4m3fn, 1024), (torch.float8_e4m3fn, 7), (torch.float8_e4m3fn, 130)])
@pytest.mark.parametrize("tokens,experts,topk,alignment", [(1, 3, 2, 1), (19, 16, 4, 1), (100, 8, 6, 128), (5, 2, 32, 16), (0, 2, 1, 1)])
def test_rows(dtype, hidden, tokens, experts, topk, alignment):
    torch.manual_seed(hidden)
    idx = _routing(tokens, experts, topk, "some masked")
    order = plan_tokens(idx.cuda(), experts, alignment=alignment)
    x = torch.randn(tokens, hidden, device="cuda").to(dtype)
    scales = torch.rand(tokens, 3, device="cuda")
    rows, row_scales = sort_tokens(x, order, scales=scales, zero_padding=True)
    raw = x.view(torch.uint8) if x.element_size() == 1 else x
    token = order.slot_map.clamp_min(0).long() // topk
    real = order.slot_map >= 0
    if tokens:
        want = torch.where(real[:, None], raw[token], torch.zeros((), dtype=raw.dtype, device="cuda"))
        assert torch.equal(rows.view(raw.dtype), want)
        assert torch.equal(row_scales, torch.where(real[:, None], scales[token], 0.0))
    assert rows.shape == (order.capacity, hidden) and row_scales.shape == (order.capacity, 3)
    again = sort_tokens(x, order)
    assert torch.equal(again.view(raw.dtype)[real], rows.view(raw.dtype)[real])


def test_rows_without_a_choice_are_left_alone():
    """The allocator gives the output the bytes of a tensor that was filled before it."""
    idx = torch.tensor([[0, -1], [2, 0], [-1, -1]], device="cuda")
    order = plan_tokens(idx, 3, alignment=4)
    x = torch.randn(3, 64, device="cuda")
    torch.cuda.synchronize()
    marked = torch.full((order.capacity, 64), 7.0, device="cuda")
    at = marked.data_ptr()
    del marked
    rows = sort_tokens(x, order)
    assert rows.data_ptr() == at
    assert bool((rows[order.slot_map < 0] == 7.0).all())


@pytest.mark.parametrize("dtype,hidden", [(torch.bfloat16, 256), (torch.bfloat16, 7168), (torch.bfloat16, 9), (torch.float16, 1000), (torch.float32, 515), (torch.float32, 512)])
@pytest.mark.parametrize("tokens,experts,topk,alignment", [(1, 3, 1, 1), (19, 16, 8, 1), (100, 8, 6, 128), (5, 2, 32, 16)])
@pytest.mark.parametrize("weighted,biased", [(True, False), (False, True), (True, True)])
def test_back(dtype, hidden, tokens, experts, topk, alignment, weighted, biased):
    torch.manual_seed(hidden)
    idx = _routing(tokens, experts, topk, "some masked")
    order = plan_tokens(idx.cuda(), experts, alignment=alignment)
    y = torch.randn(order.capacity, hidden, device="cuda").to(dtype)
    y[order.slot_map < 0] = float("nan")
    weights = torch.rand(tokens, topk, device="cuda") if weighted else None
    if weighted:
        weights[idx.cuda() < 0] = float("nan")
    bias = torch.randn(tokens, hidden, device="cuda").to(dtype) if biased else None
    out = unsort_tokens(y, order, weights, bias=bias)
    real = (order.slots >= 0)[..., None]
    terms = torch.where(real, y[order.slots.clamp_min(0).long()].double() * (weights.double()[..., None] if weighted else 1), 0.0)
    want, size = terms.sum(1), terms.abs().sum(1)
    if biased:
        want, size = want + bias.double(), size + bias.double().abs()
    assert bool(((out.double() - want).abs() <= (topk + 2) * 2.0**-24 * size + _half_step(dtype) * want.abs() * (1 + 2.0**-7) + SMALLEST[dtype]).all())


@pytest.mark.parametrize("dtype,hidden", [(torch.bfloat16, 256), (torch.bfloat16, 7168), (torch.bfloat16, 9), (torch.float16, 1000), (torch.float32, 515)])
@pytest.mark.parametrize("tokens,experts,topk,alignment", [(1, 3, 1, 1), (19, 16, 8, 1), (100, 8, 6, 128), (5, 2, 32, 16)])
def test_gradients(dtype, hidden, tokens, experts, topk, alignment):
    torch.manual_seed(hidden)
    idx = _routing(tokens, experts, topk, "some masked")
    order = plan_tokens(idx.cuda(), experts, alignment=alignment)
    real, token = order.slot_map >= 0, order.slot_map.clamp_min(0).long() // topk
    x = torch.randn(tokens, hidden, device="cuda").to(dtype).requires_grad_()
    y = torch.randn(order.capacity, hidden, device="cuda").to(dtype)
    y[~real] = float("nan")
    y.requires_grad_()
    weights = torch.rand(tokens, topk, device="cuda", requires_grad=True)
    bias = torch.randn(tokens, hidden, device="cuda").to(dtype).requires_grad_()
    g_rows = torch.randn(order.capacity, hidden, device="cuda").to(dtype)
    g_rows[~real] = float("nan")
    g_out = torch.randn(tokens, hidden, device="cuda").to(dtype)
    rows, out = sort_tokens(x, order), unsort_tokens(y, order, weights, bias=bias)
    dx, dy, dw, db = torch.autograd.grad((rows, out), (x, y, weights, bias), (g_rows, g_out))
    with torch.no_grad():
        taken = torch.where((order.slots >= 0)[..., None], g_rows[order.slots.clamp_min(0).long()].double(), 0.0)
        want, size = taken.sum(1), taken.abs().sum(1)
        assert bool(((dx.double() - want).abs() <= (topk + 1) * 2.0**-24 * size + _half_step(dtype) * want.abs() * (1 + 2.0**-7) + SMALLEST[dtype]).all())
        # one product in 32 bits, rounded to the rows' type: the same operations in torch give the same bits
        want = torch.where(real[:, None], (g_out.float()[token] * weights.flatten()[order.slot_map.clamp_min(0).long()][:, None]).to(dtype), torch.zeros((), dtype=dtype, device="cuda"))
        assert torch.equal(dy, want)
        terms = torch.where((order.slots >= 0)[..., None], y[order.slots.clamp_min(0).long()].double() * g_out.double()[:, None], 0.0)
        # eight products at a time in 32 bits, those sums in 64, one rounding
        assert bool(((dw.double() - terms.sum(-1)).abs() <= 8 * 2.0**-24 * terms.abs().sum(-1) + 2.0**-24 * terms.sum(-1).abs()).all())
        assert bool((dw[order.slots < 0] == 0).all()) and torch.equal(db, g_out)
        assert torch.equal(sort_tokens_grad(g_rows, order), dx)
        explicit = unsort_tokens_grad(g_out, y, order, weights)
        assert torch.equal(explicit[0], dy) and torch.equal(explicit[1], dw), "the same sums on every run"
        plain = unsort_tokens_grad(g_out, y, order)
        assert plain[1] is None and torch.equal(plain[0], torch.where(real[:, None], g_out[token], torch.zeros((), dtype=dtype, device="cuda")))


def test_gradients_against_differences():
    """The operators are linear in rows and bilinear in rows and weights: a difference has no error but the rounding of the forward, (K + 2) * 2^-24
    of the sizes added up, over the step."""
    torch.manual_seed(3)
    idx = _routing(6, 4, 3, "some masked").cuda()
    order = plan_tokens(idx, 4)
    x, w = torch.randn(6, 40, device="cuda"), torch.rand(6, 3, device="cuda")
    g = torch.randn(6, 40, device="cuda")

    def out(x, w):
        return unsort_tokens(sort_tokens(x, order, zero_padding=True), order, w)

    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    dx, dw = torch.autograd.grad(out(*leaves), leaves, g)
    for grad, moved in ((dx, lambda d: (x + d, w)), (dw, lambda d: (x, w + d))):
        d = torch.randn_like(grad)
        slope = (((out(*moved(d)).double() - out(*moved(-d)).double()) / 2) * g).sum()
        size = (out(x.abs() + d.abs() if grad is dx else x.abs(), w if grad is dx else w + d.abs()).double() * g.abs()).sum()
        assert abs(float(slope - (grad.double() * d.double()).sum())) <= 64 * 2.0**-24 * float(size) + 2.0**-20 * float((grad * d).abs().sum())


def test_gradients_of_some_inputs_and_once():
    order = plan_tokens(_routing(9, 4, 2, "uniform").cuda(), 4)
    y, w, b, g = torch.randn(order.capacity, 32, device="cuda"), torch.rand(9, 2, device="cuda"), torch.randn(9, 32, device="cuda"), torch.randn(9, 32, device="cuda")
    full = unsort_tokens_grad(g, y, order, w)
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((y, w, b))]
        out = unsort_tokens(leaves[0], order, leaves[1], bias=leaves[2])
        for i, grad in zip(wanted, torch.autograd.grad(out, [leaves[i] for i in wanted], g)):
            assert torch.equal(grad, (*full, g)[i])
    x, leaf = torch.randn(9, 32, device="cuda", requires_grad=True), y.clone().requires_grad_()
    for out, of in ((sort_tokens(x, order), x), (unsort_tokens(leaf, order), leaf)):
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(out.sum(), of, create_graph=True)


def test_an_expert_id_out_of_range_is_masked_and_reported():
    idx = torch.tensor([[0, 5], [7, 1], [-2, 2]], device="cuda")
    order = plan_tokens(idx, 4)
    assert order.slots.tolist() == [[0, -1], [-1, 1], [-1, 2]] and order.expert_counts.tolist() == [1, 1, 1, 0]
    with pytest.raises(RuntimeError, match="expert id"):
        gg.check_status()
    gg.check_status()


def test_what_another_stream_reports_is_seen():
    """The check waits for every stream of the device, not for the current one alone."""
    bad, stream = torch.tensor([[9]], device="cuda"), torch.cuda.Stream()
    plan_tokens(torch.tensor([[0]], device="cuda"), 4)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(200_000_000)
        plan_tokens(bad, 4)
    with pytest.raises(RuntimeError, match="expert id"):
        gg.check_status()
    gg.check_status()


def test_the_first_call_of_a_device_does_not_clear_what_the_next_one_reports(monkeypatch):
    monkeypatch.setattr(gg, "_status", {})
    good, bad, streams = torch.tensor([[0]], device="cuda"), torch.tensor([[9]], device="cuda"), [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        torch.cuda._sleep(200_000_000)
        plan_tokens(good, 4)
    with torch.cuda.stream(streams[1]):
        plan_tokens(bad, 4)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="expert id"):
        gg.check_status()


def test_captured_and_replayed():
    torch.manual_seed(0)
    idx = _routing(50, 8, 4, "some masked").cuda()
    x, w = torch.randn(50, 256, device="cuda").to(torch.bfloat16), torch.rand(50, 4, device="cuda")
    plan_tokens(idx, 8)  # the status word of the device exists from here on

    def step():
        order = plan_tokens(idx, 8, alignment=16)
        rows = sort_tokens(x, order, zero_padding=True)
        return order, rows, unsort_tokens(rows, order, w), unsort_tokens_grad(x, rows, order, w)[1], sort_tokens_grad(rows, order)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2):
        idx.copy_(_routing(50, 8, 4, "skewed", seed))
        x.normal_()
        graph.replay()
        for a, b in zip((*held[0], *held[1:]), (lambda s: (*s[0], *s[1:]))(step())):
            assert torch.equal(a, b)


def test_no_gradient_inside_a_capture():
    idx = torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    x = torch.randn(2, 16, device="cuda", requires_grad=True)
    order = plan_tokens(idx, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = torch.zeros(1, device="cuda")
        with pytest.raises(RuntimeError, match="sort_tokens_grad"):
            sort_tokens(x, order)
        with pytest.raises(RuntimeError, match="unsort_tokens_grad"):
            unsort_tokens(x, order)
    del keep


def test_another_stream_and_two_calls_at_once():
    torch.manual_seed(0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    idxs = [_routing(300, 16, 4, "uniform", s).cuda() for s in range(2)]
    x = torch.randn(300, 512, device="cuda")
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for stream, idx in zip(streams, idxs):
            with torch.cuda.stream(stream):
                order = plan_tokens(idx, 16)
                got.append((idx, order, sort_tokens(x, order)))
    torch.cuda.synchronize()
    for idx, order, rows in got:
        assert torch.equal(order.slots.cpu(), _order(idx.cpu(), 16, 1)[0])
        assert torch.equal(rows, x[order.slot_map.long() // 4])


def test_refusals():
    idx = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    order = plan_tokens(idx, 3)
    x = torch.randn(4, 64, device="cuda")
    y = torch.randn(order.capacity, 64, device="cuda")
    w = torch.rand(4, 2, device="cuda")
    for bad in (
        lambda: plan_tokens(idx.int(), 3),
        lambda: plan_tokens(idx.t(), 3),
        lambda: plan_tokens(idx, 0),
        lambda: plan_tokens(idx, 1025),
        lambda: plan_tokens(idx, 3, alignment=0),
        lambda: plan_tokens(torch.zeros(2, 33, dtype=torch.int64, device="cuda"), 64),
        lambda: sort_tokens(x[:3], order),
        lambda: sort_tokens(x.t(), order),
        lambda: sort_tokens(x.double(), order),
        lambda: sort_tokens(x, order, scales=torch.rand(3, 1, device="cuda")),
        lambda: unsort_tokens(y[:-1], order),
        lambda: unsort_tokens(y.to(torch.float8_e4m3fn), order),
        lambda: unsort_tokens(y, order, w.half()),
        lambda: unsort_tokens(y, order, w[:, :1]),
        lambda: unsort_tokens(y, order, bias=x.half()),
        lambda: unsort_tokens_grad(x.half(), y, order),
        lambda: unsort_tokens_grad(x[:2], y, order),
    ):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        plan_tokens(idx.cpu(), 3)
    with pytest.raises(ValueError):
        sort_tokens(x.requires_grad_(), order, scales=torch.rand(4, 1, device="cuda"))
