"""Operators on packed blocks: RMS norm into Q8_0 blocks, routing to experts, and products of
packed weights with Q8_0 activations.

The next step after quantizing: a layer whose weights stay packed. `rms_norm_q8` makes the
8-bit activations, `route` and `expert_plan` choose and group the experts, `matmul` and
`matmul_experts` multiply. Everything runs on the current stream of the operands' device;
outputs and workspaces are new tensors, so calls may be captured into a CUDA graph (after a
first call on the device outside of a capture, which prepares it). Nothing here is differentiable: outputs
are cut from the graph, also where an input requires a gradient. A kernel whose bounded waits run
out leaves NaN and sets the word that `_native.device_fault` reads.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch

from ._native import QS_EINVAL, SRC_IDS, QsError, block_info, check, lib

Q8_0 = 8
_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"max": 0, "top2": 1}


def _stream(index: int) -> int:
    """Handle of a device's current stream (looked up per call: a torch built without CUDA has no such function)."""
    return torch._C._cuda_getCurrentRawStream(index)


def _bad(msg: str) -> None:
    raise QsError(QS_EINVAL, msg)


def _cuda(t: torch.Tensor, what: str, index: int | None = None) -> int:
    """Index of the device of t, a CUDA tensor (on device `index`)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _bad(f"{what} must be a CUDA tensor; qsb200 runs on CUDA devices only")
    i = t.get_device()
    if index is not None and i != index:
        _bad(f"{what} is on cuda:{i}, the call runs on cuda:{index}")
    return i


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t itself if its rows start on 16-byte boundaries, else a contiguous copy."""
    n, k = t.shape
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (n <= 1 or (t.stride(0) >= k and t.stride(0) * t.element_size() % 16 == 0)):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _row_stride(t: torch.Tensor) -> int:
    """Elements between rows (of a single row: any that fits)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def rms_norm_q8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                total: torch.Tensor | None = None):
    """RMS norm of the rows of x (n, k), k a multiple of 32, into Q8_0 blocks.

    t = x + residual in x's dtype (t = x without a residual); y = t * weight / sqrt(mean(t^2) + eps).
    Returns the (n, k / 32 * 34) uint8 blocks of y, or (blocks, t) with a residual. x and
    residual: float32 / float16 / bfloat16 of one dtype; weight: k finite float32; total: where
    to write t (may be x or residual themselves), else a new tensor. Rows with inf or NaN
    decode to NaN.
    """
    dev = _cuda(x, "x")
    if not (x.dtype in SRC_IDS and x.dim() == 2):
        _bad("x must be a 2-D float32 / float16 / bfloat16 tensor")
    n, k = x.shape
    if not (k > 0 and k % 32 == 0):
        _bad(f"row length {k} is not a positive multiple of 32")
    _cuda(weight, "weight", dev)
    if not (weight.dtype == torch.float32 and weight.dim() == 1 and weight.shape[0] == k):
        _bad(f"weight must be {k} float32 values")
    weight = weight.contiguous()
    if weight.data_ptr() % 16:
        weight = weight.clone()
    src = _rows16(x)
    res = None
    if residual is not None:
        _cuda(residual, "residual", dev)
        if not (residual.dtype == x.dtype and residual.shape == x.shape):
            _bad("residual must have x's dtype and shape")
        res = _rows16(residual)
        if total is None:
            total = torch.empty((n, k), dtype=x.dtype, device=x.device)
        _cuda(total, "total", dev)
        if not (total.dtype == x.dtype and total.shape == x.shape and total.stride(1) == 1 and total.data_ptr() % 16 == 0
                and (n <= 1 or (total.stride(0) >= k and total.stride(0) * x.element_size() % 16 == 0))):
            _bad("total must have x's dtype and shape, and rows that start on 16-byte boundaries")
    elif total is not None:
        _bad("total needs a residual")
    out = torch.empty((n, k // 32 * 34), dtype=torch.uint8, device=x.device)
    check(lib().qs_rms_norm_q8(src.data_ptr(), SRC_IDS[x.dtype], _row_stride(src),
                               None if res is None else res.data_ptr(), 0 if res is None else _row_stride(res),
                               None if res is None else total.data_ptr(), 0 if res is None else _row_stride(total),
                               weight.data_ptr(), float(eps), n, k, out.data_ptr(), out.shape[1], _stream(dev)))
    return out if residual is None else (out, total)


def route(logits: torch.Tensor, top_k: int, score: str = "softmax", bias: torch.Tensor | None = None, n_groups: int = 1,
          groups_kept: int = 1, group_score: str = "max", renormalize: bool = True,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The top_k experts of every row of logits (n, experts), best first, and their weights.

    Chosen by softmax or sigmoid score + bias (float32, for the choice alone), from the
    groups_kept best of n_groups equal runs of experts (a group counts as its best expert, or as
    the sum of its two best: group_score "max" / "top2"; for the latter groups have two experts at
    least, and those with fewer than two that can be chosen come last); ties go to the lowest expert. Weights
    are the scores, over their sum if renormalize, times scale. Experts at -inf or NaN are
    never chosen; a slot left over has id -1 and weight 0. Returns ((n, top_k) int32, (n, top_k) float32).
    """
    dev = _cuda(logits, "logits")
    if not (logits.dtype in SRC_IDS and logits.dim() == 2):
        _bad("logits must be a 2-D float32 / float16 / bfloat16 tensor")
    if not (score in _SCORES):
        _bad(f"score {score!r} is not one of {list(_SCORES)}")
    if not (group_score in _GROUP_SCORES):
        _bad(f"group_score {group_score!r} is not one of {list(_GROUP_SCORES)}")
    n, e = logits.shape
    if e and (logits.stride(1) != 1 or (n > 1 and logits.stride(0) < e)):
        logits = logits.contiguous()
    if bias is not None:
        _cuda(bias, "bias", dev)
        if not (bias.dtype == torch.float32 and bias.dim() == 1 and bias.shape[0] == e):
            _bad(f"bias must be {e} float32 values")
        bias = bias.contiguous()
    top_k = int(top_k)
    ids = torch.empty((n, max(top_k, 0)), dtype=torch.int32, device=logits.device)
    weights = torch.empty((n, max(top_k, 0)), dtype=torch.float32, device=logits.device)
    check(lib().qs_route(logits.data_ptr(), SRC_IDS[logits.dtype], _row_stride(logits), n, e, top_k, _SCORES[score],
                         None if bias is None else bias.data_ptr(), int(n_groups), int(groups_kept),
                         _GROUP_SCORES[group_score], int(bool(renormalize)), float(scale), ids.data_ptr(),
                         weights.data_ptr(), _stream(dev)))
    return ids, weights


@dataclass(frozen=True)
class ExpertPlan:
    """Slots grouped by expert (expert_plan): what matmul_experts needs of a routing."""

    ids: torch.Tensor    # (tokens, top_k) int32
    table: torch.Tensor  # int32: order, then offsets
    n_experts: int

    @property
    def order(self) -> torch.Tensor:
        """(tokens * top_k,) slots by expert, those without one last."""
        return self.table[:self.ids.numel()]

    @property
    def offsets(self) -> torch.Tensor:
        """(experts + 1,): where each expert's slots start in `order`, and where the last begin."""
        return self.table[self.ids.numel():]


def expert_plan(ids: torch.Tensor, n_experts: int) -> ExpertPlan:
    """Group the slots of ids (tokens, top_k) int32 by expert; ids outside [0, n_experts) are
    slots without an expert. The plan keeps ids: do not change them while it is in use."""
    dev = _cuda(ids, "ids")
    if ids.dtype != torch.int32 or ids.dim() != 2:
        _bad("ids must be a (tokens, top_k) int32 tensor")
    ids = ids.contiguous()
    n, e = ids.numel(), int(n_experts)
    table = torch.empty(n + max(e, 0) + 1, dtype=torch.int32, device=ids.device)
    at = table.data_ptr()
    check(lib().qs_expert_plan(ids.data_ptr(), n, e, at, at + 4 * n, _stream(dev)))
    return ExpertPlan(ids, table, e)


def _packed_args(blocks: torch.Tensor, ggml_type: int, x_q8: torch.Tensor, dims: int, out_dtype: torch.dtype) -> tuple[int, int]:
    """Checks shared by the products; (device index, row length k)."""
    dev = _cuda(blocks, "blocks")
    if blocks.dtype != torch.uint8 or blocks.dim() != dims or blocks.stride(-1) != 1:
        _bad(f"blocks must be a {dims}-D uint8 tensor with packed rows in its last dimension")
    qk, nb = block_info(ggml_type)
    if min(blocks.shape) < 1 or blocks.shape[-1] % nb:
        _bad(f"weights of shape {tuple(blocks.shape)} are not rows of whole {nb}-byte blocks")
    k = blocks.shape[-1] // nb * qk
    _cuda(x_q8, "x_q8", dev)
    if x_q8.dtype != torch.uint8 or x_q8.dim() != 2 or x_q8.stride(1) != 1 or x_q8.shape[1] != k // 32 * 34:
        _bad(f"x_q8 must be row-major (rows, {k // 32 * 34}) uint8 Q8_0 blocks, as many values as the weight rows have")
    if out_dtype not in SRC_IDS:
        _bad(f"unsupported output dtype {out_dtype}")
    return dev, k


@functools.lru_cache(maxsize=1024)
def _matmul_workspace(*sizes: int) -> int:
    out = ctypes.c_int64()
    check(lib().qs_matmul_workspace(*sizes, ctypes.byref(out)))
    return out.value


@functools.lru_cache(maxsize=1024)
def _experts_workspace(*sizes: int) -> int:
    out = ctypes.c_int64()
    check(lib().qs_matmul_experts_workspace(*sizes, ctypes.byref(out)))
    return out.value


def matmul(blocks: torch.Tensor, ggml_type: int, x_q8: torch.Tensor, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """(rows, n) products of packed weights (n, row bytes) with Q8_0 activations (rows, k / 32 * 34):
    the decoded activations times the decoded weights transposed. Levels are multiplied exactly, scales
    and sums are float32, rounded once to out_dtype. For bfloat16 results of more than 32 rows the activations
    may be rounded to 11 bits first (at most 2^-11 of a value, 1/8 of the result's own rounding), and Q6_K's
    products of level and sub-scale above 2048 as well. Of many rows activations far below their row's largest are
    held to 2^-39 of 128 times the row's largest scale. The last bits of a row's result depend on the number of
    rows beside it (matmul_experts: per expert, on average), which decides the kernel; the same call gives the same
    bits every time. Row strides may exceed the rows; weight rows must start on multiples of 16 bytes for
    Q4_K / Q5_K, 8 for Q5_1 / IQ4_XS, 4 for Q4_1 / Q2_K, 2 for the others.
    """
    dev, k = _packed_args(blocks, ggml_type, x_q8, 2, out_dtype)
    n, rows = blocks.shape[0], x_q8.shape[0]
    size = _matmul_workspace(int(ggml_type), n, k, rows, SRC_IDS[out_dtype])
    out = torch.empty((rows, n), dtype=out_dtype, device=blocks.device)
    ws = torch.empty(size, dtype=torch.uint8, device=blocks.device) if size else None
    check(lib().qs_matmul(int(ggml_type), blocks.data_ptr(), _row_stride(blocks), n, k, x_q8.data_ptr(), _row_stride(x_q8), rows,
                          out.data_ptr(), SRC_IDS[out_dtype], n, None if ws is None else ws.data_ptr(), size, _stream(dev)))
    return out


def matmul_experts(blocks: torch.Tensor, ggml_type: int, x_q8: torch.Tensor, plan: ExpertPlan,
                   weights: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Products of each token with the packed weights (experts, n, row bytes) of its experts.

    x_q8: one Q8_0 row per token, or per slot (token * top_k + j). Without weights: (tokens, top_k, n),
    zeros where a slot has no expert. With weights (tokens, top_k) float32: (tokens, n), the sum of
    weight * product over a token's slots that have an expert. Otherwise as matmul; long batches take a workspace
    of 2 bytes (float32 and float16 results: 4) per slot and activation, and 4 per slot and output with weights.
    """
    dev, k = _packed_args(blocks, ggml_type, x_q8, 3, out_dtype)
    experts, n, _ = blocks.shape
    if experts != plan.n_experts:
        _bad(f"the plan is for {plan.n_experts} experts, the weights have {experts}")
    tokens, top_k = plan.ids.shape
    slots, rows = tokens * top_k, x_q8.shape[0]
    _cuda(plan.ids, "the plan", dev)
    if rows != tokens and rows != slots:
        _bad(f"x_q8 must have {tokens} or {slots} rows")
    if weights is not None:
        _cuda(weights, "weights", dev)
        if weights.dtype != torch.float32 or weights.shape != plan.ids.shape:
            _bad("weights must be (tokens, top_k) float32")
        weights = weights.contiguous()
    shape = (tokens, top_k, n) if weights is None else (tokens, n)
    if slots == 0:
        return torch.zeros(shape, dtype=out_dtype, device=blocks.device)
    row = blocks.stride(1) if n > 1 else blocks.shape[2]  # whole blocks: as aligned as the format asks
    expert = blocks.stride(0) if experts > 1 else n * row
    per_slot, summed = int(rows != tokens), int(weights is not None)
    size = _experts_workspace(int(ggml_type), experts, n, k, tokens, top_k, per_slot, summed, SRC_IDS[out_dtype])
    out = torch.empty(shape, dtype=out_dtype, device=blocks.device)
    ws = torch.empty(size, dtype=torch.uint8, device=blocks.device) if size else None
    order = plan.table.data_ptr()
    check(lib().qs_matmul_experts(int(ggml_type), blocks.data_ptr(), row, expert, experts, n, k, x_q8.data_ptr(), _row_stride(x_q8),
                                  per_slot, plan.ids.data_ptr(), order, order + 4 * slots, tokens, top_k,
                                  weights.data_ptr() if summed else None, out.data_ptr(), SRC_IDS[out_dtype], n,
                                  None if ws is None else ws.data_ptr(), size, _stream(dev)))
    return out
