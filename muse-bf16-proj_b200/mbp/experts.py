"""The rows of a mixture-of-experts layer, after ``route``: a selection sorted by expert, the tokens' rows in that
order and back, and the gradients of both directions (no counterpart in the reference, which stops at the router's
logits).

    w, ids = mbp.route(data, state, k)                  # router weights and experts of each token
    plan = mbp.expert_sort(ids, experts)                # where each assignment's row goes
    xs = mbp.expert_gather(x, plan)                     # [m*k, d]: the tokens' rows, expert by expert
    ys = mbp.expert_linear(up, xs, plan, activation="silu")   # each expert's product (mbp.linear)
    out = mbp.expert_combine(ys, w, plan, residual=x)   # [m, d]

and, for training, ``expert_combine_grad`` and ``expert_gather_grad``.  Rows are BF16 or FP32, sums FP32; every call
is one launch on the current stream of the tensors' device, uses no atomics (repeated calls give identical bits), needs no
workspace and can be captured in a CUDA graph.  Router weights and ids whose strides the kernels do not take are copied
first.  The gradients are those of the row movements; the products in between have none here (their weights are packed for
serving): a program that trains the experts brings its own product from dys to dxs.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ._lib import check, lib
from .ops import _stream

MAX_EXPERTS = 1024
_ROWS = (torch.bfloat16, torch.float32)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


@dataclass
class ExpertPlan:
    """Where the assignments of m tokens to k experts each go (assignment i = t*k + j)."""
    pos: torch.Tensor      # int32 [m, k]: row of each assignment in expert order, -1 where it was dropped
    src: torch.Tensor      # int32 [m*k]: assignment of each row, -1 past the last one
    offsets: torch.Tensor  # int32 [experts + 1]: first row of each expert; offsets[experts] rows are in use

    def __post_init__(self):
        pos, src, offsets = self.pos, self.src, self.offsets
        if pos.dtype != torch.int32 or src.dtype != torch.int32 or offsets.dtype != torch.int32:
            raise ValueError("pos, src and offsets must be int32 tensors")
        if pos.dim() != 2 or src.dim() != 1 or offsets.dim() != 1 or src.shape[0] != pos.numel() or offsets.shape[0] < 2:
            raise ValueError(f"expected pos [m, k], src [m*k] and offsets [experts + 1], got {tuple(pos.shape)}, "
                             f"{tuple(src.shape)} and {tuple(offsets.shape)}")
        if not (pos.is_contiguous() and src.is_contiguous() and offsets.is_contiguous()):
            raise ValueError("pos, src and offsets must be contiguous")
        if not pos.is_cuda or src.device != pos.device or offsets.device != pos.device:
            raise ValueError("pos, src and offsets must be CUDA tensors on one device")

    @property
    def m(self) -> int:
        return self.pos.shape[0]

    @property
    def k(self) -> int:
        return self.pos.shape[1]

    @property
    def experts(self) -> int:
        return self.offsets.shape[0] - 1


def launch(dev: torch.device, what: str, *args) -> None:
    """Calls `what`(*args, stream) with `dev` current, on its current stream; raises MbpError on a refusal."""
    if dev.index == _current_device():
        rc = getattr(lib(), what)(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = getattr(lib(), what)(*args, _stream(dev))
    if rc:
        check(rc, what)


def check_rows(t: torch.Tensor, name: str, rows: int, cols: int, dtype: torch.dtype, dev: torch.device) -> int:
    """The elements from one row of `t` to the next, once it is a [rows, cols] matrix of `dtype` on `dev` whose rows are
    contiguous and do not overlap."""
    if t.dtype is dtype and t.shape == (rows, cols) and t.device == dev:
        if t.is_contiguous():
            return cols
        ld = row_stride(t)
        if (t.stride(1) == 1 or cols == 1) and ld >= cols:
            return ld
        raise ValueError(f"{name} must have contiguous, separate rows (strides {t.stride()})")
    raise ValueError(f"{name} must be a {dtype} [{rows}, {cols}] tensor on {dev}, got {t.dtype} {list(t.shape)} on "
                     f"{t.device}")


def row_stride(t: torch.Tensor) -> int:
    """Elements from one row of a matrix to the next (a single row's stride says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the spans of memory of two tensors meet."""
    def end(t):
        return t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    return a.numel() > 0 and b.numel() > 0 and a.data_ptr() < end(b) and b.data_ptr() < end(a)


def same_rows(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices are the same elements, so that one may be written where the other is read."""
    return a.data_ptr() == b.data_ptr() and a.dtype == b.dtype and (a.stride(0) == b.stride(0) or a.shape[0] == 1)


def _check_out(out: torch.Tensor, rows: int, cols: int, like: torch.Tensor, inputs,
               in_place: torch.Tensor | None = None) -> int:
    ld = check_rows(out, "out", rows, cols, like.dtype, like.device)
    for t in inputs:
        if overlap(out, t):
            raise ValueError("out overlaps an input")
    if in_place is not None and overlap(out, in_place) and not same_rows(out, in_place):
        raise ValueError("out overlaps the residual without being the same rows")
    return ld


def _matrix(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda or t.dim() != 2 or t.dtype not in _ROWS:
        raise ValueError(f"{name} must be a 2-D bf16 or float32 CUDA tensor, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _weights(w: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    if w.dtype != torch.float32 or w.shape != plan.pos.shape or w.device != plan.pos.device:
        raise ValueError(f"weights must be a float32 {list(plan.pos.shape)} tensor on {plan.pos.device}, got {w.dtype} "
                         f"{list(w.shape)} on {w.device}")
    return w if w.is_contiguous() else w.contiguous()


def expert_sort(ids: torch.Tensor, experts: int) -> ExpertPlan:
    """The assignments ids[t][j] (int32 or int64 [m, k], rows of any stride) sorted by expert, each expert's in
    ascending t*k + j.  An id outside [0, experts) is dropped: it gets no row (pos = -1).  experts <= 1024."""
    if not ids.is_cuda or ids.dim() != 2 or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be a 2-D int32 or int64 CUDA tensor, got {ids.dtype} {tuple(ids.shape)} on {ids.device}")
    m, k = ids.shape
    if ids.is_contiguous():
        ld = k
    else:
        if k > 1 and ids.stride(1) != 1 or m > 1 and ids.stride(0) < k:
            ids = ids.contiguous()
        ld = row_stride(ids)
    dev = ids.device
    if ld == k and ids.dtype is torch.int32:
        pos = torch.empty_like(ids)
    else:
        pos = torch.empty((m, k), dtype=torch.int32, device=dev)
    src = pos.new_empty(m * k)
    offsets = pos.new_empty(experts + 1 if 0 < experts <= MAX_EXPERTS else 2)
    launch(dev, "mbp_expert_sort", ids.data_ptr(), ids.dtype is torch.int64, m, k, ld, experts, pos.data_ptr(),
           src.data_ptr(), offsets.data_ptr())
    plan = ExpertPlan.__new__(ExpertPlan)  # (what __post_init__ checks holds by construction)
    plan.pos, plan.src, plan.offsets = pos, src, offsets
    return plan


def expert_gather(x: torch.Tensor, plan: ExpertPlan, out: torch.Tensor | None = None) -> torch.Tensor:
    """xs [m*k, d]: xs[pos[t][j]] = x[t].  Rows past the last one in use are zero in a new tensor and left as they
    were in `out`."""
    _matrix(x, "x")
    m, k = plan.pos.shape
    d = x.shape[1]
    dev = plan.pos.device
    ldx = check_rows(x, "x", m, d, x.dtype, dev)
    new = out is None
    if new:
        out, ldo = x.new_empty((m * k, d)), d
    else:
        ldo = _check_out(out, m * k, d, x, (x, plan.pos, plan.offsets))
    launch(dev, "mbp_expert_gather", x.data_ptr(), x.dtype is torch.float32, m, k, d, ldx, plan.pos.data_ptr(),
           plan.offsets.data_ptr(), plan.experts, out.data_ptr(), ldo, new)
    return out


def expert_gather_grad(dxs: torch.Tensor, plan: ExpertPlan, out: torch.Tensor | None = None) -> torch.Tensor:
    """dx [m, d], the gradient of ``expert_gather``: dx[t] = sum_j dxs[pos[t][j]] (dropped assignments add nothing)."""
    return _combine(dxs, None, plan, None, out, "dxs")


def expert_combine(ys: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan, residual: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """out [m, d]: residual[t] + sum_j weights[t][j] * ys[pos[t][j]], summed in FP32 and rounded once.  Dropped
    assignments add nothing, whatever their weight.  `out` may be `residual` itself; over any other operand it is refused."""
    return _combine(ys, _weights(weights, plan), plan, residual, out, "ys")


def _combine(ys, weights, plan, residual, out, name):
    _matrix(ys, name)
    m, k = plan.pos.shape
    d, dtype, dev = ys.shape[1], ys.dtype, plan.pos.device
    ldy = check_rows(ys, name, m * k, d, dtype, dev)
    ldr = 0 if residual is None else check_rows(residual, "residual", m, d, dtype, dev)
    if out is None:
        out, ldo = ys.new_empty((m, d)), d
    else:
        ldo = _check_out(out, m, d, ys, (ys, plan.pos) if weights is None else (ys, plan.pos, weights), residual)
    launch(dev, "mbp_expert_combine", ys.data_ptr(), dtype is torch.float32, m, k, d, ldy, plan.pos.data_ptr(),
           None if weights is None else weights.data_ptr(), None if residual is None else residual.data_ptr(), ldr,
           out.data_ptr(), ldo)
    return out


def expert_combine_grad(dout: torch.Tensor, ys: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan,
                        out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(dys [m*k, d], dweights float32 [m, k]), the gradients of ``expert_combine``: dys[pos[t][j]] = weights[t][j] *
    dout[t] and dweights[t][j] = <dout[t], ys[pos[t][j]]> (0 where dropped); the residual's gradient is dout itself.
    Rows of dys past the last one in use are zero in a new tensor and left as they were in `out`."""
    _matrix(ys, "ys")
    weights = _weights(weights, plan)
    m, k = plan.pos.shape
    d = ys.shape[1]
    dev = plan.pos.device
    ldy = check_rows(ys, "ys", m * k, d, ys.dtype, dev)
    ldd = check_rows(dout, "dout", m, d, ys.dtype, dev)
    new = out is None
    if new:
        out, ldo = ys.new_empty((m * k, d)), d
    else:
        ldo = _check_out(out, m * k, d, ys, (ys, dout, weights, plan.pos, plan.offsets))
    dw = weights.new_empty((m, k))
    launch(dev, "mbp_expert_combine_grad", dout.data_ptr(), ldd, ys.data_ptr(), ldy, weights.data_ptr(),
           ys.dtype is torch.float32, m, k, d, plan.pos.data_ptr(), plan.offsets.data_ptr(), plan.experts, out.data_ptr(),
           ldo, dw.data_ptr(), new)
    return out, dw
