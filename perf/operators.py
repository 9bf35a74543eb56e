"""Performance cases of the operators around 8-bit experts: norm, token order and block-scaled products.

Four kinds of case, all on one GPU:

``norm``     ``rms_norm``: the residual's addition, the norm, and its rows in 16 bits and in e4m3 with a scale for each 128
             columns; in training its gradients.
``tokens``   ``plan_tokens``, ``sort_tokens`` and ``unsort_tokens``: a batch sorted by expert and the expert outputs summed back
             with the gate weights; in training their gradients.
``product``  ``grouped_gemm_fp8``: e4m3 rows against e4m3 expert weights with a scale for each block of 128, plain or with SwiGLU.
``block``    ``QuantizedMoE``: all of them in the order in which a model's layer runs them.

``own`` selects the framework's kernels; without it the operators are computed in elementary torch operations.
"""

from __future__ import annotations

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST, BLOCK, TINY, EPS = 448.0, 128, 1e-30, 1e-6

# ----------------------------------------------------------------------------------------------- cases


def _norm(name, tokens, hidden, *, dtype="bf16", residual=True, quantize=True, keep=True, train=False):
    return dict(name=name, kind="norm", tokens=tokens, hidden=hidden, dtype=dtype, residual=residual, quantize=quantize, keep=keep, train=train)


def _tokens(name, tokens, hidden, experts, topk, *, dtype="e4m3", routing="balanced", alignment=1, bias=False, train=False):
    return dict(name=name, kind="tokens", tokens=tokens, hidden=hidden, experts=experts, topk=topk, dtype=dtype, routing=routing,
                alignment=alignment, bias=bias, train=train)


def _product(name, tokens, k, n, experts, topk, *, swiglu=False, quantize=False, scaled=False, routing="balanced"):
    return dict(name=name, kind="product", tokens=tokens, k=k, n=n, experts=experts, topk=topk, swiglu=swiglu,
                quantize=quantize, scaled=scaled, routing=routing)


def _block(name, tokens, hidden, inner, experts, topk, routing="balanced"):
    return dict(name=name, kind="block", tokens=tokens, hidden=hidden, inner=inner, experts=experts, topk=topk, routing=routing)


def listed():
    return [
        # The norm in front of an expert layer, one sequence in decode: latency.
        _norm("norm-1", 1, 7168),
        # The same for a prefill chunk: memory traffic.
        _norm("norm-4096", 4096, 7168),
        # A training step's norm on a ragged batch, forward and gradients (rows kept in 16 bits).
        _norm("norm-train-3001", 3001, 4096, quantize=False, train=True),
        # A decode batch to and from the experts, rows in 8 bits with their scales.
        _tokens("tokens-32", 32, 7168, 256, 8),
        # A prefill chunk of the same.
        _tokens("tokens-4096", 4096, 7168, 256, 8),
        # A training step on a ragged batch with uneven experts: rows in 16 bits, padded for the 16-bit GEMM, and all gradients.
        _tokens("tokens-train-3001", 3001, 4096, 64, 6, dtype="bf16", routing="zipf", alignment=128, train=True),
        # A dense layer of one sequence in decode (one matrix, one row): latency and weight traffic.
        _product("product-1", 1, 7168, 4096, 1, 1),
        # Up-projection of one GPU's 32 of 256 experts in a decode step: weight traffic.
        _product("product-decode-64", 512, 7168, 4096, 32, 1, swiglu=True, quantize=True),
        # Down-projection with uneven experts and an inner size that is no multiple of 1024, gate weights applied.
        _product("product-down-777", 777, 1536, 4096, 32, 6, scaled=True, routing="zipf"),
        # Up-projection of the same 32 experts in prefill: tensor cores.
        _product("product-prefill-4096", 4096, 7168, 4096, 32, 8, swiglu=True, quantize=True),
        # A whole layer with 64 small experts in a decode step.
        _block("block-32", 32, 4096, 1536, 64, 6),
        # The same layer on a mid-sized batch with uneven experts.
        _block("block-1000", 1000, 4096, 1536, 64, 6, routing="zipf"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the same ranges; never more work than the largest listed case of its kind."""
    kind = rng.choice(["norm", "tokens", "product", "product", "block"])
    routing = rng.choice(["balanced", "uniform", "zipf"])
    if kind == "norm":
        hidden = rng.choice([8 * rng.randint(16, 1024), 256 * rng.randint(1, 32), rng.randint(100, 8192)])
        train = rng.random() < 0.35
        quantize = not train and rng.random() < 0.7
        case = _norm("", _log_int(rng, 1, 4096 * 7168 // max(hidden, 7168)), hidden, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                     residual=rng.random() < 0.7, quantize=quantize, keep=not quantize or rng.random() < 0.5, train=train)
    elif kind == "tokens":
        experts = rng.choice([4, 8, 32, 60, 64, 128, 160, 256, 512])
        topk = rng.randint(1, min(8, experts))
        train = rng.random() < 0.4
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"]) if train or rng.random() < 0.3 else "e4m3"
        hidden = rng.choice([256 * rng.randint(2, 28), 8 * rng.randint(20, 900), rng.randint(150, 7168)])
        tokens = _log_int(rng, 1, min(4096, 3001 * 4096 * 6 // (hidden * topk)))
        case = _tokens("", tokens, hidden, experts, topk, dtype=dtype, routing=routing, alignment=rng.choice([1, 1, 16]), bias=rng.random() < 0.3, train=train)
    elif kind == "product":
        swiglu = rng.random() < 0.5
        k, n = rng.choice([128 * rng.randint(2, 56), 16 * rng.randint(8, 448)]), rng.choice([256 * rng.randint(1, 28), 32 * rng.randint(4, 200)])
        experts = rng.choice([1, 1, 4, 8, 16, 24, 32])
        topk = rng.randint(1, min(8, experts))
        tokens = _log_int(rng, 1, min(8192, 4096 * 8 * 7168 * 4096 // (topk * k * n)))
        case = _product("", tokens, k, n, experts, topk, swiglu=swiglu, quantize=swiglu and rng.random() < 0.7,
                        scaled=not swiglu and rng.random() < 0.5, routing=routing)
    else:
        hidden, inner = 256 * rng.randint(4, 28), 128 * rng.randint(4, 16)
        experts = rng.choice([8, 16, 32])
        topk = rng.randint(1, 8)
        case = _block("", _log_int(rng, 1, min(2048, 1000 * 6 * 4096 * 1536 // (topk * hidden * inner))), hidden, inner, experts, topk, routing=routing)
    del case["name"]
    return case


# ----------------------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _routing(gen, tokens, experts, topk, kind, masked=True):
    """A router's softmax top-k (balanced), uniformly random experts, or experts of Zipf(1.2) popularity, with a tenth of the
    choices after the first masked (unless every choice has to count)."""
    if kind == "balanced":
        w, idx = torch.softmax(torch.randn(tokens, experts, generator=gen, device="cuda"), dim=-1).topk(topk, dim=-1)
        return idx, w / w.sum(-1, keepdim=True)
    if kind == "uniform":
        idx = torch.rand(tokens, experts, generator=gen, device="cuda").topk(topk, dim=-1).indices
        return idx, torch.full((tokens, topk), 1.0 / topk, device="cuda")
    popularity = torch.arange(1, experts + 1, device="cuda").float().pow(-1.2)[torch.randperm(experts, generator=gen, device="cuda")]
    noise = torch.rand(tokens, experts, generator=gen, device="cuda").clamp_(1e-12, 1 - 1e-7).log().neg().log().neg()
    idx = (popularity.log() + noise).topk(topk, dim=-1).indices
    w = torch.rand(tokens, topk, generator=gen, device="cuda") + 0.1
    drop = torch.rand(tokens, topk, generator=gen, device="cuda") < 0.1
    drop[:, 0] = False
    return idx.masked_fill(drop & masked, -1), w / w.sum(-1, keepdim=True)


def _activations(gen, rows, columns):
    """e4m3 rows with a scale for each 128 columns, from values whose size differs from row to row."""
    return _quantize(torch.randn(rows, columns, generator=gen, device="cuda") * torch.exp(torch.randn(rows, 1, generator=gen, device="cuda")))


def _weights(gen, experts, rows, columns, halves=1):
    """e4m3 weights ``[experts, rows, columns]`` with a scale for each 128 x 128 block of each half."""
    part, down, across = rows // halves, -(-rows // halves // BLOCK), -(-columns // BLOCK)
    q = torch.empty(experts, rows, columns, dtype=E4M3, device="cuda")
    scales = torch.empty(experts, halves * down, across, device="cuda")
    for e in range(experts):
        for h in range(halves):
            w = torch.randn(part, columns, generator=gen, device="cuda") * (0.02 * (1 + torch.rand(1, generator=gen, device="cuda")))
            blocks = torch.nn.functional.pad(w, (0, across * BLOCK - columns, 0, down * BLOCK - part)).view(down, BLOCK, across, BLOCK)
            s = blocks.abs().amax((1, 3)).clamp_min(TINY) / LARGEST
            q[e, h * part : (h + 1) * part] = (blocks / s[:, None, :, None]).reshape(down * BLOCK, -1)[:part, :columns].to(E4M3)
            scales[e, h * down : (h + 1) * down] = s
    return q, scales


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": case}
    if case["kind"] == "norm":
        t, h, dtype = case["tokens"], case["hidden"], TYPES[case["dtype"]]
        state["x"] = _normal(gen, t, h, dtype=dtype)
        state["weight"] = _normal(gen, h, scale=0.2, dtype=dtype) + 1
        state["residual"] = _normal(gen, t, h, scale=3.0, dtype=dtype) if case["residual"] else None
        if case["train"]:
            state["grad_y"] = _normal(gen, t, h, dtype=dtype)
            state["grad_residual"] = _normal(gen, t, h, dtype=dtype) if case["residual"] else None
    elif case["kind"] == "tokens":
        t, h, topk = case["tokens"], case["hidden"], case["topk"]
        state["idx"], state["gate"] = _routing(gen, t, case["experts"], topk, case["routing"])
        dtype = TYPES.get(case["dtype"], torch.bfloat16)
        if case["dtype"] == "e4m3":
            state["x"], state["scales"] = _activations(gen, t, h)
        else:
            state["x"], state["scales"] = _normal(gen, t, h, dtype=dtype), None
        state["y"] = _normal(gen, _capacity(case), h, dtype=dtype)
        state["bias"] = _normal(gen, t, h, dtype=dtype) if case["bias"] else None
        if case["train"]:
            state["grad_rows"], state["grad_out"] = _normal(gen, _capacity(case), h, dtype=dtype), _normal(gen, t, h, dtype=dtype)
    elif case["kind"] == "product":
        idx, _ = _routing(gen, case["tokens"], case["experts"], case["topk"], case["routing"], masked=False)
        counts = (idx.flatten()[:, None] == torch.arange(case["experts"], device="cuda")).sum(0)
        rows = int(counts.sum())
        state["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        state["most"] = int(counts.max())
        state["a"], state["a_scales"] = _activations(gen, rows, case["k"])
        state["w"], state["w_scales"] = _weights(gen, case["experts"], case["n"], case["k"], 2 if case["swiglu"] else 1)
        state["row_scale"] = torch.rand(rows, generator=gen, device="cuda") if case["scaled"] else None
        # rows of each expert side by side, for the plain form's batched product
        state["at"] = state["offsets"][:-1, None] + torch.arange(state["most"], device="cuda")
        state["real"] = torch.arange(state["most"], device="cuda") < counts[:, None]
    else:
        t, h, inner, experts = case["tokens"], case["hidden"], case["inner"], case["experts"]
        state["idx"], state["gate"] = _routing(gen, t, experts, case["topk"], case["routing"])
        state["x"], state["residual"] = _normal(gen, t, h), _normal(gen, t, h, scale=3.0)
        state["weight"] = _normal(gen, h, scale=0.2) + 1
        state["w13"], state["s13"] = _weights(gen, experts, 2 * inner, h, 2)
        state["w2"], state["s2"] = _weights(gen, experts, h, inner)
        state["most"] = int((state["idx"].flatten()[:, None] == torch.arange(experts, device="cuda")).sum(0).max())
    return state


# ----------------------------------------------------------------------------------------------- plain forms


def _capacity(case):
    """Rows that hold every choice of the batch, whatever the routing."""
    choices, a = case["tokens"] * case["topk"], case.get("alignment", 1)
    return -(-(choices + min(case["experts"], choices) * (a - 1)) // a) * a


def _quantize(v, factor=None):
    """Rows ``v * factor`` (a factor for each row) -> e4m3 rows and a scale for each 128 columns.  The factor is not needed for the
    e4m3 values: many of them lie on the border of two (products of two 16-bit values over another one), in 64 bits exactly."""
    rows, n = v.shape
    across = -(-n // BLOCK)
    blocks = torch.nn.functional.pad(v.double(), (0, across * BLOCK - n)).view(rows, across, BLOCK)
    most = blocks.abs().amax(-1).clamp_min(TINY)
    q = (blocks * LARGEST / most[..., None]).view(rows, -1)[:, :n].to(E4M3)
    return q, (most / LARGEST if factor is None else most * factor / LARGEST).float()


def _dequantize(q, scales):
    return q.float() * scales.repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _plain_norm(x, weight, residual):
    """The residual stream in its type, its product with the weight and what the norm scales it by."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    return h, h.double() * weight.double(), torch.rsqrt(h.float().square().mean(-1, keepdim=True) + EPS)


def _plain_order(idx, experts, alignment, capacity):
    """Stable order of the choices by expert: slot of each choice, choice of each slot, counts and offsets."""
    flat = idx.reshape(-1)
    key = torch.where(flat >= 0, flat, experts)
    perm = torch.argsort(key, stable=True)
    counts = (key[:, None] == torch.arange(experts, device=key.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), ((counts + alignment - 1) // alignment * alignment).cumsum(0)])
    first = torch.cat([counts.new_zeros(1), counts.cumsum(0)])  # of each expert in the order without gaps
    ordered = key[perm]
    slot = torch.where(ordered < experts, offsets[ordered] + torch.arange(len(key), device=key.device) - first[ordered], capacity)
    slot_map = torch.full((capacity + 1,), -1, dtype=torch.int32, device=key.device)
    slot_map[slot] = perm.int()
    slots = torch.empty_like(key)
    slots[perm] = torch.where(slot < capacity, slot, -1)
    return slots.view(idx.shape).int(), slot_map[:capacity], counts, offsets


def _plain_sort(x, slot_map, topk):
    rows = x.view(torch.uint8) if x.dtype == E4M3 else x
    rows = torch.where(slot_map[:, None] >= 0, rows[slot_map.clamp_min(0).long() // topk], torch.zeros((), dtype=rows.dtype, device=x.device))
    return rows.view(x.dtype)


def _plain_unsort(y, slots, gate, bias):
    rows = torch.where(slots[..., None] >= 0, y[slots.clamp_min(0).long()].float(), 0.0)
    out = (rows if gate is None else rows * gate[..., None]).sum(1)
    return (out if bias is None else out + bias.float()).to(y.dtype)


def _plain_product(a, w, w_scales, at, real, swiglu):
    """fp32 rows against every expert's weights, as one batched product over the experts' rows side by side."""
    experts, n, k = w.shape
    halves = 2 if swiglu else 1
    s = w_scales.view(experts * halves, -1, w_scales.shape[-1]).repeat_interleave(BLOCK, 1)[:, : n // halves].repeat_interleave(BLOCK, 2)[..., :k]
    w = w.float() * s.reshape(experts, n, k)
    y = torch.bmm(a[at.clamp_max(len(a) - 1)], w.transpose(1, 2))
    if swiglu:
        gate, up = y.chunk(2, -1)
        y = gate / (1 + torch.exp(-gate)) * up
    out = torch.zeros(len(a) + 1, y.shape[-1], device=a.device)
    out[torch.where(real, at, len(a))] = y
    return out[:-1]


def _plain_norm_case(s):
    case = s["case"]
    h, v, rstd = _plain_norm(s["x"], s["weight"], s["residual"])
    out = {"residual": h} if case["residual"] else {}
    if case["keep"]:
        out["y"] = (v.float() * rstd).to(h.dtype)
    if case["quantize"]:
        out["q"], out["scales"] = _quantize(v, rstd)
    if case["train"]:
        xhat, g = h.float() * rstd, s["grad_y"].float()
        gw = g * s["weight"].float()
        dx = rstd * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
        out["dx"] = (dx if s["grad_residual"] is None else dx + s["grad_residual"].float()).to(h.dtype)
        out["dweight"] = (g * xhat).sum(0, dtype=torch.float64).to(h.dtype)
    return out


def _plain_tokens_case(s):
    case, topk = s["case"], s["case"]["topk"]
    slots, slot_map, counts, offsets = _plain_order(s["idx"], case["experts"], case["alignment"], _capacity(case))
    out = dict(slots=slots, slot_map=slot_map, counts=counts, offsets=offsets, rows=_plain_sort(s["x"], slot_map, topk),
               out=_plain_unsort(s["y"], slots, s["gate"], s["bias"]))
    if s["scales"] is not None:
        out["row_scales"] = _plain_sort(s["scales"], slot_map, topk)
    if case["train"]:
        g, token, real = s["grad_out"].float(), slot_map.clamp_min(0).long() // topk, slot_map[:, None] >= 0
        out["dx"] = _plain_unsort(s["grad_rows"], slots, None, None)
        out["dy"] = torch.where(real, g[token] * s["gate"].reshape(-1)[slot_map.clamp_min(0).long()][:, None], 0.0).to(s["y"].dtype)
        dots = (s["y"][slots.clamp_min(0).long()].float() * g[:, None]).sum(-1, dtype=torch.float64)
        out["dgate"] = torch.where(slots >= 0, dots, 0.0).float()
        if s["bias"] is not None:
            out["dbias"] = s["grad_out"]
    return out


def _plain_product_case(s):
    case = s["case"]
    y = _plain_product(_dequantize(s["a"], s["a_scales"]), s["w"], s["w_scales"], s["at"], s["real"], case["swiglu"])
    if s["row_scale"] is not None:
        y = y * s["row_scale"][:, None]
    if case["quantize"]:
        q, scales = _quantize(y)
        return {"q": q, "scales": scales}
    return {"out": y.to(torch.bfloat16)}


def _plain_block_case(s):
    case, topk = s["case"], s["case"]["topk"]
    h, v, rstd = _plain_norm(s["x"], s["weight"], s["residual"])
    q, scales = _quantize(v, rstd)
    capacity = _capacity(case)
    slots, slot_map, counts, offsets = _plain_order(s["idx"], case["experts"], 1, capacity)
    a = _dequantize(_plain_sort(q, slot_map, topk), _plain_sort(scales, slot_map, topk))
    at = offsets[:-1, None] + torch.arange(s["most"], device=a.device)
    real = torch.arange(s["most"], device=a.device) < counts[:, None]
    inner = _dequantize(*_quantize(_plain_product(a, s["w13"], s["s13"], at, real, True)))
    rows = _plain_product(inner, s["w2"], s["s2"], at, real, False).to(torch.bfloat16)
    return {"out": _plain_unsort(rows, slots, s["gate"], None), "residual": h}


# ----------------------------------------------------------------------------------------------- one pass


def _own_norm(s):
    from nanoep_b200.ops.rms_norm import rms_norm

    case = s["case"]
    if not case["train"]:
        got = rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, quantize=case["quantize"], keep=case["keep"])
        out = {"residual": got.residual} if case["residual"] else {}
        if case["keep"]:
            out["y"] = got.y
        if case["quantize"]:
            out["q"], out["scales"] = got.q, got.scales
        return out
    x, weight = s["x"].detach().requires_grad_(), s["weight"].detach().requires_grad_()
    got = rms_norm(x, weight, residual=s["residual"], eps=EPS)
    if not case["residual"]:
        dx, dweight = torch.autograd.grad(got.y, (x, weight), s["grad_y"])
        return {"y": got.y, "dx": dx, "dweight": dweight}
    dx, dweight = torch.autograd.grad((got.y, got.residual), (x, weight), (s["grad_y"], s["grad_residual"]))
    return {"residual": got.residual, "y": got.y, "dx": dx, "dweight": dweight}


def _own_tokens(s):
    from nanoep_b200.ops.token_order import plan_tokens, sort_tokens, unsort_tokens

    case = s["case"]
    order = plan_tokens(s["idx"], case["experts"], alignment=case["alignment"])
    out = dict(slots=order.slots, slot_map=order.slot_map, counts=order.expert_counts, offsets=order.expert_offsets)
    if not case["train"]:
        rows = sort_tokens(s["x"], order, scales=s["scales"], zero_padding=True)
        if s["scales"] is not None:
            rows, out["row_scales"] = rows
        return dict(out, rows=rows, out=unsort_tokens(s["y"], order, s["gate"], bias=s["bias"]))
    x, y, gate = (s[name].detach().requires_grad_() for name in ("x", "y", "gate"))
    bias = None if s["bias"] is None else s["bias"].detach().requires_grad_()
    rows = sort_tokens(x, order, zero_padding=True)
    back = unsort_tokens(y, order, gate, bias=bias)
    leaves = (x, y, gate) if bias is None else (x, y, gate, bias)
    grads = torch.autograd.grad((rows, back), leaves, (s["grad_rows"], s["grad_out"]))
    out.update(rows=rows, out=back, dx=grads[0], dy=grads[1], dgate=grads[2])
    if bias is not None:
        out["dbias"] = grads[3]
    return out


def _own_product(s):
    from nanoep_b200.ops.fp8_gemm import grouped_gemm_fp8

    case = s["case"]
    got = grouped_gemm_fp8(s["a"], s["a_scales"], s["w"], s["w_scales"], s["offsets"], swiglu=case["swiglu"], quantize=case["quantize"],
                           row_scale=s["row_scale"], max_expert_rows=s["most"])
    return {"q": got[0], "scales": got[1]} if case["quantize"] else {"out": got}


def _own_block(s):
    from nanoep_b200.models.quantized_moe import QuantizedMoE

    if "layer" not in s:  # a model keeps it
        s["layer"] = QuantizedMoE(s["w13"], s["s13"], s["w2"], s["s2"], norm_weight=s["weight"], eps=EPS)
    out, residual = s["layer"](s["x"], s["idx"], s["gate"], residual=s["residual"])
    return {"out": out, "residual": residual}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "tokens": _own_tokens, "product": _own_product, "block": _own_block}[kind](state)
    return {"norm": _plain_norm_case, "tokens": _plain_tokens_case, "product": _plain_product_case, "block": _plain_block_case}[kind](state)


# ----------------------------------------------------------------------------------------------- work


def _expected_experts(case):
    """Experts that get at least one row, in expectation."""
    choices = case["tokens"] * case["topk"]
    return case["experts"] * (1 - (1 - 1 / case["experts"]) ** choices) if case["experts"] > 1 else 1


def _scale_bytes(rows, columns):
    return rows * -(-columns // BLOCK) * 4


def work(case):
    if case["kind"] == "norm":
        t, h, size = case["tokens"], case["hidden"], TYPES[case["dtype"]].itemsize
        row = h * size
        per = row * ((3 if case["residual"] else 1) + (1 if case["keep"] else 0)) + (h + _scale_bytes(1, h) if case["quantize"] else 0)
        flops = 8 * t * h
        if case["train"]:
            per += row * (3 if case["residual"] else 2)
            flops += 14 * t * h
        return {"bytes": t * per + row * (2 if case["train"] else 1), "flops": flops}
    if case["kind"] == "tokens":
        t, h, k = case["tokens"], case["hidden"], case["topk"]
        x_row = h + _scale_bytes(1, h) if case["dtype"] == "e4m3" else h * TYPES[case["dtype"]].itemsize
        y_row = h * TYPES.get(case["dtype"], torch.bfloat16).itemsize
        moved = t * x_row + t * k * x_row + t * k * y_row + t * y_row * (2 if case["bias"] else 1) + t * k * (8 + 4 + 4 + 4)
        flops = 2 * t * k * h
        if case["train"]:
            moved += t * k * x_row + t * x_row + t * y_row + 2 * t * k * y_row
            flops += 4 * t * k * h
        return {"bytes": moved, "flops": flops}
    if case["kind"] == "product":
        rows, k, n = case["tokens"] * case["topk"], case["k"], case["n"]
        wide = n // 2 if case["swiglu"] else n
        written = rows * wide + _scale_bytes(rows, wide) if case["quantize"] else 2 * rows * wide
        return {"bytes": _expected_experts(case) * n * k + rows * k + _scale_bytes(rows, k) + written, "flops": 2 * rows * n * k}
    t, h, inner, rows = case["tokens"], case["hidden"], case["inner"], case["tokens"] * case["topk"]
    return {"bytes": _expected_experts(case) * 3 * inner * h + 4 * 2 * t * h, "flops": 6 * rows * inner * h + 8 * t * h}


# ----------------------------------------------------------------------------------------------- 64 bits


def _exact_blocks(v, factor=1.0):
    """Values over the largest of their block, times 448 (a row's factor cancels), and the scales; unrounded."""
    most = torch.stack([part.abs().amax(1).clamp(min=TINY) for part in v.split(BLOCK, 1)], 1)
    return torch.cat([part * LARGEST / most[:, b : b + 1] for b, part in enumerate(v.split(BLOCK, 1))], 1), most * factor / LARGEST


def _exact_rows(q, scales):
    return torch.cat([part * scales[:, b : b + 1].double() for b, part in enumerate(q.double().split(BLOCK, 1))], 1)


def _exact_weight(w, scales):
    """One matrix, its row blocks and column blocks scaled."""
    return torch.cat([_exact_rows(part, scales[b : b + 1].expand(len(part), -1)) for b, part in enumerate(w.split(BLOCK, 0))], 0)


def _exact_expert(rows, w, scales, swiglu):
    if not swiglu:
        return rows @ _exact_weight(w, scales).T
    half, down = len(w) // 2, len(scales) // 2
    gate, up = rows @ _exact_weight(w[:half], scales[:down]).T, rows @ _exact_weight(w[half:], scales[down:]).T
    return gate * torch.sigmoid(gate) * up


def _exact_norm(x, weight, residual):
    total = x.double() if residual is None else x.double() + residual.double()
    h = total.to(x.dtype).double()  # the stream is held in its type
    rms = (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt()
    return total, h, h * weight.double(), rms


def _exact_order(idx, experts, alignment, capacity):
    choice = idx.flatten().tolist()
    counts = [0] * experts
    for e in choice:
        if e >= 0:
            counts[e] += 1
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + -(-c // alignment) * alignment)
    at, slots, slot_map = offsets[:-1].copy(), [], [-1] * capacity
    for i, e in enumerate(choice):
        slots.append(at[e] if e >= 0 else -1)
        if e >= 0:
            slot_map[at[e]] = i
            at[e] += 1
    return slots, slot_map, counts, offsets


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        total, h, v, rms = _exact_norm(s["x"], s["weight"], s["residual"])
        out = {"residual": total} if case["residual"] else {}
        if case["keep"]:
            out["y"] = v / rms
        if case["quantize"]:
            out["q"], out["scales"] = _exact_blocks(v, 1 / rms)
        if case["train"]:
            g, xhat = s["grad_y"].double(), h / rms
            gw = g * s["weight"].double()
            out["dx"] = (gw - xhat * (gw * xhat).sum(1, keepdim=True) / case["hidden"]) / rms
            if case["residual"]:
                out["dx"] = out["dx"] + s["grad_residual"].double()
            out["dweight"] = torch.einsum("th,th->h", g, xhat)
        return out
    if case["kind"] == "tokens":
        slots, slot_map, counts, offsets = (torch.tensor(v, device="cuda") for v in _exact_order(s["idx"], case["experts"], case["alignment"], _capacity(case)))
        slots, gate, y = slots.view(s["idx"].shape), s["gate"].double(), s["y"]
        out = dict(slots=slots.int(), slot_map=slot_map.int(), counts=counts, offsets=offsets)
        filled = (slot_map >= 0).nonzero().flatten()
        token = slot_map[filled] // case["topk"]

        def spread(v):
            rows = torch.zeros(len(slot_map), *v.shape[1:], dtype=torch.float64, device="cuda")
            rows[filled] = v.double()[token]
            return rows

        def back(v, weights):
            acc = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
            return acc.index_add_(0, token, v.double()[filled] * weights.flatten()[slot_map[filled]][:, None])

        out["rows"] = spread(s["x"])
        if s["scales"] is not None:
            out["row_scales"] = spread(s["scales"])
        out["out"] = back(y, gate)
        if s["bias"] is not None:
            out["out"] = out["out"] + s["bias"].double()
        if case["train"]:
            g = s["grad_out"].double()
            out["dx"] = back(s["grad_rows"], torch.ones_like(gate))
            dy, dgate = torch.zeros(y.shape, dtype=torch.float64, device="cuda"), torch.zeros(gate.numel(), dtype=torch.float64, device="cuda")
            dy[filled] = g[token] * gate.flatten()[slot_map[filled]][:, None]
            dgate[slot_map[filled]] = torch.einsum("rh,rh->r", g[token], y[filled].double())
            out.update(dy=dy, dgate=dgate.view(gate.shape))
            if s["bias"] is not None:
                out["dbias"] = g
        return out
    if work(case)["flops"] > 2e14:
        return None  # over 20 seconds in 64 bits
    if case["kind"] == "product":
        rows = _exact_rows(s["a"], s["a_scales"])
        wide = case["n"] // 2 if case["swiglu"] else case["n"]
        y = torch.zeros(len(rows), wide, dtype=torch.float64, device="cuda")
        ends = s["offsets"].tolist()
        for e in range(case["experts"]):
            if ends[e + 1] > ends[e]:
                y[ends[e] : ends[e + 1]] = _exact_expert(rows[ends[e] : ends[e + 1]], s["w"][e], s["w_scales"][e], case["swiglu"])
        if s["row_scale"] is not None:
            y = y * s["row_scale"].double()[:, None]
        if case["quantize"]:
            q, scales = _exact_blocks(y)
            return {"q": q, "scales": scales}
        return {"out": y}
    total, _, v, rms = _exact_norm(s["x"], s["weight"], s["residual"])
    q, scales = _exact_blocks(v, 1 / rms)
    rows = _exact_rows(q.to(E4M3), scales)  # held in 8 bits between the products
    out = torch.zeros_like(total)
    for e in range(case["experts"]):
        token, k = (s["idx"] == e).nonzero(as_tuple=True)
        if len(token):
            q, scales = _exact_blocks(_exact_expert(rows[token], s["w13"][e], s["s13"][e], True))
            part = _exact_expert(_exact_rows(q.to(E4M3), scales), s["w2"][e], s["s2"][e], False).to(torch.bfloat16)  # rows travel back in 16 bits
            out.index_add_(0, token, part.double() * s["gate"][token, k].double()[:, None])
    return {"out": out, "residual": total}
