"""Block-scaled product of 8-bit rows and expert weights, against 64 bits.

Tolerances.  Products of two e4m3 values are exact in 32 bits.  A sum of 128 of them, scaled, and of ceil(K / 128) such parts is a chain of at
most 128 + K / 128 + 4 roundings; a tensor core may cut instead of rounding, 2^-23 each, of the sum of the terms' sizes.  silu(gate) * up
adds 2^-18 relative (exponential, quotient, products) and passes the errors of its factors on (the slope of silu is at most 1.1).
bf16 rounds by 2^-8 at most, e4m3 by 2^-4 (2^-10 of the scale among its denormals)."""

import pytest
import torch

from nanoep_b200.ops import grouped_gemm as gg
from nanoep_b200.ops.fp8_gemm import grouped_gemm_fp8, quantize_rows, quantize_weights

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _problem(counts, K, N, *, alignment=1, swiglu=False, tail=0, seed=0, poison=True):
    """Rows of every expert, gaps and rows behind the last one hold NaN."""
    gen = torch.Generator(device="cuda").manual_seed(seed + K + N)
    ranges = [-(-c // alignment) * alignment for c in counts]
    offsets = torch.tensor([0] + ranges, device="cuda").cumsum(0)
    rows = int(offsets[-1]) + tail
    a, a_scales = quantize_rows(torch.randn(rows, K, generator=gen, device="cuda") * torch.exp(torch.randn(rows, 1, generator=gen, device="cuda")))
    real = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for e, c in enumerate(counts):
        real[int(offsets[e]) : int(offsets[e]) + c] = True
    if poison:
        a.view(torch.uint8)[~real] = 0x7F
        a_scales[~real] = float("nan")
    w = torch.randn(len(counts), N, K, generator=gen, device="cuda") * 0.05 * torch.exp(torch.randn(len(counts), N, 1, generator=gen, device="cuda"))
    q, scales = quantize_weights(w, swiglu=swiglu)
    return a, a_scales, q, scales, offsets, torch.tensor(counts, device="cuda"), real


def _spread(scales, columns):
    return scales.double().repeat_interleave(128, -1)[..., :columns]


def _reference(a, a_scales, w, w_scales, offsets, counts, swiglu, row_scale=None):
    """Result in 64 bits and a bound of its error in 32."""
    K, halves = a.shape[1], 2 if swiglu else 1
    n = w.shape[1] // halves
    rows = a.double() * _spread(a_scales, K)
    out = torch.zeros(len(a), n, dtype=torch.float64, device="cuda")
    off = torch.zeros_like(out)
    step = (128 + -(-K // 128) + 4) * 2.0**-23
    for e in range(len(w)):
        lo = int(offsets[e])
        mine = slice(lo, lo + int(counts[e]))
        if counts[e] == 0:
            continue
        full = w[e].double().view(halves, n, K) * _spread(w_scales[e].view(halves, -1, w_scales.shape[-1]).transpose(1, 2), n).transpose(1, 2).repeat_interleave(128, 2)[..., :K]
        y = [rows[mine] @ part.T for part in full]
        d = [step * (rows[mine].abs() @ part.abs().T) for part in full]
        if swiglu:
            act = y[0] * torch.sigmoid(y[0])
            out[mine] = act * y[1]
            off[mine] = 1.1 * d[0] * y[1].abs() + act.abs() * d[1] + 1.1 * d[0] * d[1] + 2.0**-18 * (act * y[1]).abs()
        else:
            out[mine], off[mine] = y[0], d[0]
    if row_scale is not None:
        out, off = out * row_scale.double()[:, None], off * row_scale.double().abs()[:, None] + 2.0**-23 * (out * row_scale.double()[:, None]).abs()
    return out, off


def _check(got, want, off, real):
    assert bool(((got.double() - want).abs()[real] <= (off + 2.0**-8 * (want.abs() + off))[real]).all())


def _check_quantized(q, scales, want, off, real):
    n = want.shape[1]
    pad = -n % 128
    most, worst = (torch.nn.functional.pad(t, (0, pad)).view(len(t), (n + pad) // 128, 128).abs().amax(-1) for t in (want, off))
    assert bool(((scales.double() - most.clamp_min(1e-30) / 448).abs()[real] <= (worst / 448 + 2.0**-22 * most / 448)[real]).all())
    value, step = q.double() * _spread(scales, n), _spread(scales, n)
    assert bool(((value - want).abs()[real] <= (off + (2.0**-4 + 2.0**-20) * (want.abs() + off) + 2.0**-10 * step + 2.0**-22 * want.abs())[real]).all())
    assert bool((torch.nn.functional.pad(q.float(), (0, pad)).view(len(q), (n + pad) // 128, 128).abs().amax(-1)[real & (most.amin(-1) > 1e-20)] == 448).all())


COUNTS = [[1], [0], [5], [64, 0, 1], [127, 128, 129], [0, 0, 257, 1, 0, 33], [700, 3], [31, 32, 33, 63, 65, 0, 96, 100, 1, 2]]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("K,N", [(128, 128), (16, 16), (144, 272), (1024, 512), (2064, 144), (640, 1040)])
@pytest.mark.parametrize("scaled", [False, True])
def test_plain(counts, K, N, scaled):
    a, sa, w, sw, offsets, n, real = _problem(counts, K, N)
    scale = torch.rand(len(a), device="cuda") + 0.5 if scaled else None
    out = grouped_gemm_fp8(a, sa, w, sw, offsets, row_scale=scale, max_expert_rows=max(counts) if scaled else 0)
    gg.check_status()
    want, off = _reference(a, sa, w, sw, offsets, n, False, scale)
    _check(out, want, off, real)


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("K,I", [(128, 128), (16, 16), (144, 272), (1024, 512), (2064, 144)])
@pytest.mark.parametrize("quantize", [False, True])
def test_swiglu(counts, K, I, quantize):
    a, sa, w, sw, offsets, n, real = _problem(counts, K, 2 * I, swiglu=True)
    got = grouped_gemm_fp8(a, sa, w, sw, offsets, swiglu=True, quantize=quantize, max_expert_rows=max(counts) if quantize else 0)
    gg.check_status()
    want, off = _reference(a, sa, w, sw, offsets, n, True)
    if quantize:
        _check_quantized(*got, want, off, real)
    else:
        _check(got, want, off, real)


@pytest.mark.parametrize("alignment,tail", [(1, 3), (16, 0), (128, 130)])
@pytest.mark.parametrize("quantize", [False, True])
def test_rows_that_do_not_exist(alignment, tail, quantize):
    """Gaps between experts, rows that an expert's count leaves out and rows behind the last hold NaN: no real row sees one, and none is written."""
    counts = [37, 0, 128, 1, 300]
    a, sa, w, sw, offsets, n, real = _problem(counts, 512, 256, alignment=alignment, tail=tail)
    for t in (torch.empty(len(a), 256, dtype=torch.bfloat16, device="cuda"), torch.empty(len(a), 256, dtype=E4M3, device="cuda")):
        t.view(torch.uint8).fill_(0x55)  # bytes that the allocator hands out again
        del t
    got = grouped_gemm_fp8(a, sa, w, sw, offsets, expert_counts=n, quantize=quantize)
    gg.check_status()
    want, off = _reference(a, sa, w, sw, offsets, n, False)
    if quantize:
        _check_quantized(*got, want, off, real)
    else:
        _check(got, want, off, real)
        assert bool((got.view(torch.uint8)[~real] == 0x55).all())
    # a count that is larger than the range, or negative, is cut to it
    more = n.clone()
    more[1], more[3] = 5, -4
    again = grouped_gemm_fp8(a, sa, w, sw, offsets, expert_counts=more, quantize=quantize)
    first = got[0] if quantize else got
    same = (again[0] if quantize else again).view(torch.uint8) == first.view(torch.uint8)
    keep = real.clone()
    keep[int(offsets[3]) : int(offsets[4])] = False
    assert bool(same[keep].all())


@pytest.mark.parametrize("counts", [[1], [16], [17, 0, 40], [129, 300, 0, 5], [33, 64, 65, 128, 256, 257]])
@pytest.mark.parametrize("tile,ctas,columns", [(32, 1, 0), (32, 2, 256), (32, 4, 256), (32, 8, 256), (64, 1, 256), (64, 2, 256), (64, 8, 256), (128, 1, 0), (32, 1, 128), (32, 4, 128),
                                               (64, 2, 128), (64, 8, 128)])
@pytest.mark.parametrize("K,n,swiglu,quantize,scaled", [(128, 48, False, False, True), (2064, 400, False, True, False), (1024, 384, True, True, False), (400, 144, True, False, False)])
def test_every_kernel(counts, tile, ctas, columns, K, n, swiglu, quantize, scaled):
    """Every tile and split of the K axis, also where a CTA's part of it is empty."""
    a, sa, w, sw, offsets, c, real = _problem(counts, K, 2 * n if swiglu else n, swiglu=swiglu, tail=2)
    scale = torch.rand(len(a), device="cuda") + 0.5 if scaled else None
    got = gg._ext().grouped_gemm_fp8(a, sa, w, sw, offsets, None, scale, swiglu, quantize, 0, gg.status_tensor(a.device), tile, ctas, columns)
    gg.check_status()
    want, off = _reference(a, sa, w, sw, offsets, c, swiglu, scale)
    if quantize:
        _check_quantized(*got, want, off, real)
    else:
        _check(got[0], want, off, real)


@pytest.mark.parametrize("K", [112, 256, 384, 1024, 1136])
@pytest.mark.parametrize("swiglu,quantize,scaled", [(False, False, False), (False, False, True), (False, True, False), (True, False, False), (True, True, False)])
def test_several_tiles_a_block(K, swiglu, quantize, scaled):
    """Rows as M on more than twice as many tiles as the GPU holds, full ones beside those of a few rows, over one to nine blocks of K."""
    n, counts = 1040, [e * 37 % 300 + 1 for e in range(40)]
    tiles = sum(-(-c // 128) for c in counts) * (-(-n // 128) if swiglu else -(-n // 256))
    assert tiles > 2 * torch.cuda.get_device_properties(0).multi_processor_count and any(c % 128 and c % 128 <= 32 for c in counts)
    a, sa, w, sw, offsets, c, real = _problem(counts, K, 2 * n if swiglu else n, swiglu=swiglu, tail=2)
    scale = torch.rand(len(a), device="cuda") + 0.5 if scaled else None
    got = gg._ext().grouped_gemm_fp8(a, sa, w, sw, offsets, None, scale, swiglu, quantize, 0, gg.status_tensor(a.device), 128, 1, 0)
    gg.check_status()
    want, off = _reference(a, sa, w, sw, offsets, c, swiglu, scale)
    if quantize:
        _check_quantized(*got, want, off, real)
    else:
        _check(got[0], want, off, real)


@pytest.mark.parametrize("tile", [32, 64, 128])
def test_exact_sums_round_as_rows_do(tile):
    """Sums of digits, exact in 32 bits: the e4m3 result is that of the quotient, ties to even, and what quantize_rows gives for the same values."""
    gen = torch.Generator(device="cuda").manual_seed(tile)
    rows, blocks = 300, 4
    m = 28 * torch.randint(1, 2341, (rows, 1), generator=gen, device="cuda")  # 448 = 16 * 28: T * m / 28 is a whole number whose quotient is T * 16
    tie = torch.randint(8, 14, (rows, 128), generator=gen, device="cuda") * 2 + 1
    v = torch.where(torch.rand(rows, 128, generator=gen, device="cuda") < 0.5, tie * m // 28, torch.randint(0, 1 << 16, (rows, 128), generator=gen, device="cuda") % (m + 1))
    v[:, 5:6] = m
    digits = torch.cat([v >> 4 * b & 15 for b in range(blocks)], 1).float().to(E4M3)
    a_scales = torch.tensor([16.0**b for b in range(blocks)], device="cuda").repeat(rows, 1)
    w = torch.eye(128, device="cuda").repeat(1, blocks)[None].to(E4M3)
    offsets = torch.tensor([0, rows], device="cuda")
    q, scales = gg._ext().grouped_gemm_fp8(digits, a_scales, w, torch.ones(1, 1, blocks, device="cuda"), offsets, None, None, False, True, 0, gg.status_tensor(w.device), tile, 1, 0)
    gg.check_status()
    want = v.double() * 448 / m
    step = torch.exp2(torch.frexp(want.clamp_min(2.0**-6)).exponent.double() - 4)
    assert torch.equal(q.double(), torch.round(want / step) * step)
    again = quantize_rows(v.float())
    assert torch.equal(q.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(scales, again[1])


@pytest.mark.parametrize("rows", [1, 3, 64, 129])
def test_one_matrix(rows):
    a, sa, w, sw, offsets, n, real = _problem([rows], 768, 384)
    out = grouped_gemm_fp8(a, sa, w[0], sw[0])
    want, off = _reference(a, sa, w, sw, offsets, n, False)
    _check(out, want, off, real)
    q = grouped_gemm_fp8(a, sa, w[0], sw[0], quantize=True)
    _check_quantized(*q, want, off, real)


@pytest.mark.parametrize("rows,K,N", [(1, 7168, 512), (2, 16384, 256), (300, 7168, 256)])
def test_a_long_axis(rows, K, N):
    a, sa, w, sw, offsets, n, real = _problem([rows], K, N)
    out = grouped_gemm_fp8(a, sa, w, sw, offsets)
    want, off = _reference(a, sa, w, sw, offsets, n, False)
    _check(out, want, off, real)
    assert torch.equal(out, grouped_gemm_fp8(a, sa, w, sw, offsets)), "the same sums on every run"


def test_many_units_and_experts():
    """More tiles than the GPU holds at a time, 300 experts, most with a few rows and some with none."""
    counts = [(e * 7) % 23 if e % 5 else 0 for e in range(300)]
    a, sa, w, sw, offsets, n, real = _problem(counts, 256, 512, swiglu=True)
    q, scales = grouped_gemm_fp8(a, sa, w, sw, offsets, swiglu=True, quantize=True)
    want, off = _reference(a, sa, w, sw, offsets, n, True)
    _check_quantized(q, scales, want, off, real)


def test_a_row_does_not_depend_on_the_others():
    """The same row alone, in a small and in a large expert, and under a hint: the order of the sums may differ with the tile, nothing else."""
    a, sa, w, sw, offsets, n, real = _problem([600], 1024, 256)
    whole = grouped_gemm_fp8(a, sa, w, sw, offsets)
    for first, last in ((0, 1), (5, 100), (128, 384), (599, 600)):
        part = grouped_gemm_fp8(a[first:last].contiguous(), sa[first:last].contiguous(), w, sw, torch.tensor([0, last - first], device="cuda"), max_expert_rows=last - first)
        torch.testing.assert_close(part.float(), whole[first:last].float(), rtol=2.0**-7, atol=1e-3)


@pytest.mark.parametrize("rows,experts,most,k_blocks", [(1, 1, 1, 56), (64, 1, 0, 16), (512, 32, 32, 56), (512, 32, 0, 56), (4096, 32, 0, 16), (40000, 32, 0, 56), (7, 256, 0, 8), (3, 3, 900, 1)])
def test_the_choice_covers_every_call(rows, experts, most, k_blocks):
    for swiglu in (False, True):
        tile, ctas, n_tiles = gg._ext().fp8_gemm_choice(rows, experts, most, 16, swiglu, k_blocks, 148)
        assert tile in (32, 64, 128) and ctas in (1, 2, 4, 8) and (tile < 128 or ctas == 1)
        assert n_tiles == 16 if swiglu else n_tiles in (8, 16) and (tile < 128 or n_tiles == 8)


def test_extreme_scales_and_values():
    """Scales far from one, blocks of zeros, infinities of a scale and NaN stay in their own rows and columns."""
    a, sa, w, sw, offsets, n, real = _problem([40], 512, 256)
    sa[3] *= 1e20
    sa[4] *= 1e-25
    sa[5, 1] = float("inf")
    a.view(torch.uint8)[6, 77] = 0x7F
    a[7] = torch.zeros(512, device="cuda").to(E4M3)
    out = grouped_gemm_fp8(a, sa, w, sw, offsets)
    want, off = _reference(a, sa, w, sw, offsets, n, False)
    assert not bool(out[5].isfinite().any()) and bool(out[6].isnan().all()) and not out[7].any()
    fine = torch.ones(40, dtype=torch.bool, device="cuda")
    fine[5] = fine[6] = False
    _check(out, want, off, fine)
    q, scales = grouped_gemm_fp8(a, sa, w, sw, offsets, quantize=True)
    assert bool(scales[6].isnan().all()) and not q[7].float().any() and bool((scales[7] > 0).all())


def test_offsets_that_fall_are_reported():
    a, sa, w, sw, offsets, n, real = _problem([10, 10], 128, 128)
    for bad in ([0, 15, 10], [1, 10, 20], [0, 10, 21], [-5, 10, 20]):
        grouped_gemm_fp8(a, sa, w, sw, torch.tensor(bad, device="cuda"))
        with pytest.raises(RuntimeError, match="expert_offsets"):
            gg.check_status()
    grouped_gemm_fp8(a, sa, w, sw, offsets)
    gg.check_status()


def test_captured_and_replayed_beside_another_graph():
    """Two graphs and an eager call on different streams share no workspace."""
    problems = [_problem(c, 7168, 256, seed=s) for s, c in enumerate(([1], [2], [3]))]
    want = [grouped_gemm_fp8(*p[:5]) for p in problems]
    graphs, held = [], []
    for p in problems[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(grouped_gemm_fp8(*p[:5]))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    eager = []
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager.append(grouped_gemm_fp8(*problems[2][:5]))
    torch.cuda.synchronize()
    assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]) and all(torch.equal(t, want[2]) for t in eager)


def test_refusals():
    a, sa, w, sw, offsets, n, real = _problem([10, 10], 256, 256)
    i64 = dict(dtype=torch.int64, device="cuda")
    for bad in (
        lambda: grouped_gemm_fp8(a.float(), sa, w, sw, offsets),
        lambda: grouped_gemm_fp8(a.t(), sa, w, sw, offsets),
        lambda: grouped_gemm_fp8(a[:, :128].contiguous(), sa, w, sw, offsets),
        lambda: grouped_gemm_fp8(a, sa[:, :1], w, sw, offsets),
        lambda: grouped_gemm_fp8(a, sa.half(), w, sw, offsets),
        lambda: grouped_gemm_fp8(a, sa, w, sw[:, :1], offsets),
        lambda: grouped_gemm_fp8(a, sa, w, sw, offsets, swiglu=True, row_scale=torch.rand(20, device="cuda")),
        lambda: grouped_gemm_fp8(a, sa, w, sw, offsets, row_scale=torch.rand(19, device="cuda")),
        lambda: grouped_gemm_fp8(a, sa, w, sw),
        lambda: grouped_gemm_fp8(a, sa, w, sw, torch.zeros(2, **i64)),
        lambda: grouped_gemm_fp8(a, sa, w, sw, offsets.int()),
        lambda: grouped_gemm_fp8(a, sa, w, sw, offsets, expert_counts=torch.zeros(3, **i64)),
        lambda: grouped_gemm_fp8(a, sa, w, sw, offsets, max_expert_rows=-1),
        lambda: grouped_gemm_fp8(a, sa, w[:, :8].contiguous(), sw[:, :1].contiguous(), offsets),
        lambda: grouped_gemm_fp8(torch.zeros(20, 8, device="cuda").to(E4M3), sa[:, :1].contiguous(), torch.zeros(2, 16, 8, device="cuda").to(E4M3), sw[:, :1, :1].contiguous(), offsets),
    ):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        grouped_gemm_fp8(a.cpu(), sa, w, sw, offsets)
    assert grouped_gemm_fp8(a[:0], sa[:0], w, sw, torch.zeros(3, **i64)).shape == (0, 256)
