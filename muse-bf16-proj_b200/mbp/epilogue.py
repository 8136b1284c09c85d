"""Projections with an epilogue, and the same product per expert (no counterpart in the reference, whose projections
return the bare product).

``linear`` computes residual + mul * activation(x @ W[:n].T + bias) in one launch on the kernels behind ``gemv``
(m <= 32 tokens) and ``gemm`` (more): the operands are added to the FP32 sums, which are rounded once.
``expert_linear`` does the same for rows sorted by expert (``expert_sort``), each segment against its own matrix of a
``PackedExperts``; the segments' borders stay on the device, so nothing waits for them on the host.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from ._lib import Epilogue
from .experts import ExpertPlan, check_rows, launch, overlap, same_rows
from .ops import BASE_TILE, PackedC12, _check_x, pack_c12, unpack_c12

ACTIVATIONS = {"none": 0, "relu": 1, "relu2": 2, "gelu": 3, "gelu_tanh": 4, "silu": 5, "sigmoid": 6}  # MBP_ACT_*
# One matrix: the GEMV up to 32 tokens, the tcgen05 GEMM above, the boundary of kernel_fn (so that both give the same bits).
# A small matrix would take the GEMM earlier: 1536 x 6144 at 24 tokens 17 us on the GEMV and 11 us there.
GEMV_MAX_M = 32
_TYPES = (torch.bfloat16, torch.float32)


@dataclass
class PackedExperts:
    """`experts` BF16 matrices of one shape [n, k], packed one after the other in the lossless 12-bit format, the
    columns of every 64-column chunk in the tensor cores' order (mbp_expert_order)."""
    packed: PackedC12  # [experts * n, k]
    experts: int

    @property
    def n(self) -> int:
        return self.packed.n // self.experts

    @property
    def k(self) -> int:
        return self.packed.k

    @property
    def nbytes(self) -> int:
        return self.packed.nbytes


def pack_experts(w: torch.Tensor, base_mode: int = BASE_TILE) -> PackedExperts:
    """Packs [experts, n, k] BF16 weights (n % 16 == 0, k % 64 == 0, experts <= 1024) on their device."""
    if not w.is_cuda or w.dtype != torch.bfloat16 or w.dim() != 3:
        raise ValueError(f"expected a 3-D bf16 CUDA tensor, got {w.dtype} {tuple(w.shape)} on {w.device}")
    e, n, k = w.shape
    if not 1 <= e <= 1024 or n < 16 or n % 16 or k < 64 or k % 64:
        raise ValueError(f"expert weights {tuple(w.shape)}: 1 to 1024 experts, rows a multiple of 16, columns of 64")
    with torch.cuda.device(w.device):
        return PackedExperts(pack_c12(_reorder(w.reshape(e * n, k), 0), base_mode), e)


def unpack_experts(p: PackedExperts) -> torch.Tensor:
    """The weights [experts, n, k], bit for bit."""
    with torch.cuda.device(p.packed.units.device):
        return _reorder(unpack_c12(p.packed), 1).view(p.experts, p.n, p.k)


def _reorder(w: torch.Tensor, back: int) -> torch.Tensor:
    w = w.contiguous()
    if w.data_ptr() % 4:
        w = w.clone()
    out = torch.empty_like(w)
    launch(w.device, "mbp_expert_order", w.data_ptr(), w.shape[0], w.shape[1], out.data_ptr(), back)
    return out


def _tokens(x: torch.Tensor, k: int, device: torch.device) -> torch.Tensor:
    if x.is_cuda and x.dim() == 2 and (not x.is_contiguous() or x.data_ptr() % 16):
        x = x.clone(memory_format=torch.contiguous_format)
    _check_x(x, k, device)
    return x


def _epilogue(m, n, dev, bias, bias_shape, activation, mul, residual):
    """The C epilogue of a call (the tensors in it have to outlive the launch)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r} (one of {', '.join(ACTIVATIONS)})")
    e = Epilogue()
    e.activation = ACTIVATIONS[activation]
    if bias is not None:
        if bias.dtype not in _TYPES or tuple(bias.shape) != bias_shape or bias.device != dev:
            raise ValueError(f"bias must be a bf16 or float32 {list(bias_shape)} tensor on {dev}, got {bias.dtype} "
                             f"{list(bias.shape)} on {bias.device}")
        bias = bias if bias.is_contiguous() else bias.contiguous()
        e.bias, e.bias_f32 = bias.data_ptr(), bias.dtype is torch.float32
    if mul is not None:
        if mul.dtype not in _TYPES:
            raise ValueError(f"mul must be bf16 or float32, got {mul.dtype}")
        e.ld_mul = check_rows(mul, "mul", m, n, mul.dtype, dev)
        e.mul, e.mul_f32 = mul.data_ptr(), mul.dtype is torch.float32
    if residual is not None:
        if residual.dtype not in _TYPES:
            raise ValueError(f"residual must be bf16 or float32, got {residual.dtype}")
        e.ld_residual = check_rows(residual, "residual", m, n, residual.dtype, dev)
        e.residual, e.residual_f32 = residual.data_ptr(), residual.dtype is torch.float32
    return e, bias


def _output(out, out_dtype, m, n, x, mul, residual, p, *others):
    """(the output tensor, its row stride)"""
    if out is None:
        if out_dtype not in _TYPES:
            raise ValueError(f"unsupported output dtype {out_dtype}")
        return (x.new_empty((m, n)) if out_dtype is x.dtype else x.new_empty((m, n), dtype=out_dtype)), n
    if out.dtype not in _TYPES:
        raise ValueError(f"unsupported output dtype {out.dtype}")
    ld = check_rows(out, "out", m, n, out.dtype, x.device)
    if ld > 0x7fffffff:
        raise ValueError("out rows are too far apart")
    for t in (x, p.units, p.bases, p.esc_off, p.esc, *others):
        if t is not None and overlap(out, t):
            raise ValueError("out overlaps x, the bias, the plan or the packed weights")
    for name, t in (("mul", mul), ("residual", residual)):
        if t is not None and overlap(out, t) and not same_rows(out, t):
            raise ValueError(f"out overlaps {name} without being the same rows")
    return out, ld


def linear(p: PackedC12, x: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none",
           mul: torch.Tensor | None = None, residual: torch.Tensor | None = None, n_out: int | None = None,
           out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """residual + mul * activation(x @ W[:n_out].T + bias): [m, n_out] in `out`'s type or `out_dtype` (bf16, float32).

    x is BF16 [m, k]; bias [n_out], mul and residual [m, n_out] (rows of any stride) are each BF16 or FP32.  `out` may
    be `mul` or `residual` itself; any other overlap with an operand is refused."""
    n = p.n if n_out is None else n_out
    x = _tokens(x, p.k, p.units.device)
    m, dev = x.shape[0], x.device
    e, bias = _epilogue(m, n, dev, bias, (n,), activation, mul, residual)
    out, ld = _output(out, out_dtype, m, n, x, mul, residual, p, bias)
    e.out_f32 = out.dtype is torch.float32
    if m > GEMV_MAX_M:
        launch(dev, "mbp_gemm_c12_epi", p.desc_ptr, x.data_ptr(), m, n, ctypes.byref(e), out.data_ptr(), ld)
    else:
        launch(dev, "mbp_gemv_c12_epi", p.desc_ptr, x.data_ptr(), m, n, ctypes.byref(e), out.data_ptr(), ld, None)
    return out


def expert_linear(p: PackedExperts, xs: torch.Tensor, plan: ExpertPlan, bias: torch.Tensor | None = None,
                  activation: str = "none", mul: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                  tensor_cores: bool | None = None, tile: int = 0) -> torch.Tensor:
    """``linear`` of each row with its own expert's matrix: row r of xs [m*k, k_in] (``expert_gather``'s order) belongs
    to the expert e with plan.offsets[e] <= r < plan.offsets[e+1].  bias is [experts, n]; mul, residual and out are by
    row.  Rows past the last one in use are zero in a new tensor and left as they were in `out`.

    Few rows per expert run on the GEMV, more on the tcgen05 GEMM (`tensor_cores` overrides); `tile` (8, 16 or 32, 0
    chooses) is the GEMV's and chooses it: rows of one expert per pass over its weights."""
    if plan.experts != p.experts:
        raise ValueError(f"plan of {plan.experts} experts, weights of {p.experts}")
    xs = _tokens(xs, p.k, p.packed.units.device)
    rows, dev, n = xs.shape[0], xs.device, p.n
    if rows != plan.src.shape[0] or dev != plan.offsets.device:
        raise ValueError(f"xs must have the plan's {plan.src.shape[0]} rows on {plan.offsets.device}, got {rows} on {dev}")
    e, bias = _epilogue(rows, n, dev, bias, (p.experts, n), activation, mul, residual)
    new = out is None
    out, ld = _output(out, out_dtype, rows, n, xs, mul, residual, p.packed, bias, plan.offsets)
    e.out_f32 = out.dtype is torch.float32
    if tile:
        if tensor_cores:
            raise ValueError("tile is the GEMV's: not with tensor_cores=True")
        tensor_cores = False
    elif tensor_cores is None:
        tensor_cores = _use_tensor_cores(rows, p)
    args = (p.packed.desc_ptr, p.experts, xs.data_ptr(), rows, plan.offsets.data_ptr(), ctypes.byref(e), new,
            out.data_ptr(), ld)
    if tensor_cores:
        launch(dev, "mbp_gemm_c12_experts", *args)
    else:
        launch(dev, "mbp_gemv_c12_experts", *args, tile)
    return out


def _use_tensor_cores(rows: int, p: PackedExperts) -> bool:
    """Measured, GEMV / GEMM in us.  Selections with popular and unused experts, 64 of them: at 8 and 10 rows per expert on
    average 161 / 163 and 170 / 164 (1536 x 6144), 174 / 184 and 191 / 185 (6144 x 1536); of 512 x 1024, whose 50 MB the GEMV
    streams in less than the GEMM's fixed cost, 16.3 / 20.5 at 12 and 21.4 / 21.0 at 16.  As many rows for each: 64 of
    1536 x 6144 153 / 195 at 8 and 177 / 196 at 12, 256 of them 601 / 675 and 702 / 682.  Not measured: a few experts, and
    one that takes most of the rows."""
    per = 16 if p.packed.n * p.k <= 64 << 20 else 8
    return rows > per * p.experts
