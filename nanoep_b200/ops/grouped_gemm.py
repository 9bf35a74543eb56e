"""Grouped GEMM over expert-major rows (tcgen05 / TMEM kernels, csrc/expert_gemm_sm100.cu; gated by row counters:
csrc/grouped_gemm_sm100.cu and its CTA-pair variant).

``rows`` come from a dispatch with ``do_expand=True, alignment=128``: every 128-row block belongs to one expert.  Padding rows
may hold anything (``expert_counts`` says how many rows of an expert exist) unless row blocks are gated by counters, which
count them too (``zero_padding=True``).  The reference library stops at
dispatch/combine; these ops are the expert compute that sits between them on the same GPU.
"""

from __future__ import annotations

import threading

import torch

PLAIN, SWIGLU = 0, 1
_status: dict[int, torch.Tensor] = {}
_status_lock = threading.Lock()


def _ext():
    from ..utils.build import load_extension

    return load_extension()


def status_tensor(device) -> torch.Tensor:
    index = torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    if index not in _status:
        with _status_lock:
            if index not in _status:
                made = torch.zeros(4, dtype=torch.int32, device=torch.device("cuda", index))
                if not torch.cuda.is_current_stream_capturing():
                    torch.cuda.current_stream(index).synchronize()  # kernels on other streams write to it as well, from the next call on
                _status[index] = made
    return _status[index]


def operator_status(x: torch.Tensor) -> torch.Tensor:
    """``status_tensor`` of a tensor's device for operators that can be captured: it must exist before a capture starts."""
    found = _status.get(x.device.index) if x.is_cuda else None
    if found is not None:
        return found
    if not x.is_cuda:
        raise ValueError("operands must be CUDA tensors")
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the first call on a device cannot be captured: call once before the capture, as for any warm-up")
    return status_tensor(x.device)


def refuse_captured_gradients(name: str, explicit: str):
    """Autograd's accumulation nodes remember the stream of the graph that made them; one that outlives into a capture ends the process.
    The explicit gradient functions have no such nodes."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name} is not differentiated inside a CUDA graph capture: call {explicit} there")


def refuse_gradients(name: str, *tensors):
    """For operators without a gradient: a result that is cut off from autograd's graph looks like one that depends on less than it does."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{name} has no gradient and got a tensor that requires one: call it under torch.no_grad(), or with detached tensors")


def check_status(device=None):
    """Raise if a kernel of these operators on ``device`` gave up on a bounded wait or met invalid indices.  Waits for the device, all its streams."""
    st = status_tensor(device if device is not None else torch.cuda.current_device())
    torch.cuda.synchronize(st.device)
    code, cta = (int(v) for v in st[:2].tolist())
    if code != 0:
        st.zero_()
        torch.cuda.synchronize(st.device)  # what another stream reports from here on stays
        reasons = {101: "an operand pipeline wait timed out", 102: "the wait for a row block's ready counter timed out",
                   103: "expert_offsets are not multiples of 128 from 0 to the row count", 104: "handle metadata names an impossible rank, token or row",
                   105: "an expert id lies outside [-1, num_experts)", 106: "expert_offsets fall, do not start at 0 or end behind the rows"}
        raise RuntimeError(f"nanoep_b200 grouped GEMM status {code} ({reasons.get(code, 'unknown')}), detail {cta}")


def grouped_gemm(a, w, expert_offsets, *, swiglu: bool = False, out=None, tile_ready=None, tile_expected=None, max_ctas: int = 0,
                 timeout_s: float = 5.0, row_scale=None, stages: int = 4, pair: bool = False, expert_counts=None, max_expert_rows: int = 0) -> torch.Tensor:
    """``out[r] = a[r] @ w[e(r)].T`` (bf16 in, fp32 accumulate, bf16 out).

    a: ``[rows, K]`` bf16, rows % 128 == 0;  w: ``[E, N, K]`` bf16 (``[E, 2*I, K]`` gate rows then up
    rows when ``swiglu``);  expert_offsets: int64 ``[E+1]`` row offsets (multiples of 128).
    With ``swiglu`` the result is ``silu(a @ w_gate.T) * (a @ w_up.T)`` of shape ``[rows, I]``.
    ``row_scale`` (fp32 ``[rows]``, plain mode) multiplies each output row in FP32 before the bf16 round.
    ``expert_counts`` (int64 ``[E]``): only so many rows of each expert's range exist; the other rows are neither read as
    far as the result goes nor defined in the output.  ``max_expert_rows`` (0 = unknown): no expert holds more rows.
    It has no gradient: autograd sees its result as a constant.
    ``stages=3`` runs the single-CTA kernel with a pipeline that leaves a third of an SM's shared memory to another kernel,
    ``pair=True`` the CTA-pair kernel (two SMs share every weight tile); both compute every row of every range, and they are
    what runs with ``tile_ready`` (row blocks gated by counters).
    """
    n_out = w.shape[1] // 2 if swiglu else w.shape[1]
    if out is None:
        out = torch.empty((a.shape[0], n_out), dtype=torch.bfloat16, device=a.device)
    _ext().grouped_gemm(a, w, expert_offsets, out, status_tensor(a.device), SWIGLU if swiglu else PLAIN, tile_ready, tile_expected,
                        int(max_ctas), float(timeout_s), row_scale, int(stages), bool(pair), expert_counts, int(max_expert_rows))
    return out


def grouped_gemm_reference(a, w, expert_offsets, *, swiglu: bool = False) -> torch.Tensor:
    """Plain PyTorch fp32 reference of the same op (for tests)."""
    offsets = expert_offsets.tolist()
    n_out = w.shape[1] // 2 if swiglu else w.shape[1]
    out = torch.zeros((a.shape[0], n_out), dtype=torch.float32, device=a.device)
    for e in range(w.shape[0]):
        lo, hi = offsets[e], offsets[e + 1]
        if hi <= lo:
            continue
        y = a[lo:hi].float() @ w[e].float().t()
        if swiglu:
            inner = w.shape[1] // 2
            y = torch.nn.functional.silu(y[:, :inner]) * y[:, inner:]
        out[lo:hi] = y
    return out
