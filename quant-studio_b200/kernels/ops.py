"""Operators on packed blocks: RMS norm into Q8_0 blocks, routing to experts, and products of
packed weights with Q8_0 activations.

The next step after quantizing: a layer whose weights stay packed. `rms_norm_q8` makes the
8-bit activations, `route` and `expert_plan` choose and group the experts, `matmul` and
`matmul_experts` multiply. Everything runs on the current stream of the operands' device;
outputs and workspaces are new tensors, so calls may be captured into a CUDA graph.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from ._native import QS_EINVAL, SRC_IDS, QsError, block_info, check, lib

Q8_0 = 8
_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"max": 0, "top2": 1}


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise QsError(QS_EINVAL, msg)


def _cuda(t: torch.Tensor, what: str, device: torch.device | None = None) -> None:
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise QsError(QS_EINVAL, f"{what} must be a CUDA tensor; qsb200 runs on CUDA devices only")
    if device is not None and t.device != device:
        raise QsError(QS_EINVAL, f"{what} is on {t.device}, the call runs on {device}")


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t itself if its rows start on 16-byte boundaries, else a contiguous copy."""
    n, k = t.shape
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (n <= 1 or (t.stride(0) >= k and t.stride(0) * t.element_size() % 16 == 0)):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def rms_norm_q8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                total: torch.Tensor | None = None):
    """RMS norm of the rows of x (n, k), k a multiple of 32, into Q8_0 blocks.

    t = x + residual in x's dtype (t = x without a residual); y = t * weight / sqrt(mean(t^2) + eps).
    Returns the (n, k / 32 * 34) uint8 blocks of y, or (blocks, t) with a residual. x and
    residual: float32 / float16 / bfloat16 of one dtype; weight: k finite float32; total: where
    to write t (may be x or residual themselves), else a new tensor. Rows with inf or NaN
    decode to NaN.
    """
    _cuda(x, "x")
    _need(x.dtype in SRC_IDS and x.dim() == 2, "x must be a 2-D float32 / float16 / bfloat16 tensor")
    n, k = x.shape
    _need(k > 0 and k % 32 == 0, f"row length {k} is not a positive multiple of 32")
    _cuda(weight, "weight", x.device)
    _need(weight.dtype == torch.float32 and weight.dim() == 1 and weight.shape[0] == k, f"weight must be {k} float32 values")
    weight = weight.contiguous()
    if weight.data_ptr() % 16:
        weight = weight.clone()
    src = _rows16(x)
    res = None
    if residual is not None:
        _cuda(residual, "residual", x.device)
        _need(residual.dtype == x.dtype and residual.shape == x.shape, "residual must have x's dtype and shape")
        res = _rows16(residual)
        if total is None:
            total = torch.empty((n, k), dtype=x.dtype, device=x.device)
        _cuda(total, "total", x.device)
        _need(total.dtype == x.dtype and total.shape == x.shape and total.stride(1) == 1 and total.data_ptr() % 16 == 0
              and (n <= 1 or (total.stride(0) >= k and total.stride(0) * x.element_size() % 16 == 0)),
              "total must have x's dtype and shape, and rows that start on 16-byte boundaries")
    else:
        _need(total is None, "total needs a residual")
    out = torch.empty((n, k // 32 * 34), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().qs_rms_norm_q8(src.data_ptr(), SRC_IDS[x.dtype], _row_stride(src),
                                   None if res is None else res.data_ptr(), 0 if res is None else _row_stride(res),
                                   None if res is None else total.data_ptr(), 0 if res is None else _row_stride(total),
                                   weight.data_ptr(), float(eps), n, k, out.data_ptr(), out.shape[1], _stream(x.device)))
    return out if residual is None else (out, total)


def route(logits: torch.Tensor, top_k: int, score: str = "softmax", bias: torch.Tensor | None = None, n_groups: int = 1,
          groups_kept: int = 1, group_score: str = "max", renormalize: bool = True,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The top_k experts of every row of logits (n, experts), best first, and their weights.

    Chosen by softmax or sigmoid score + bias (float32, for the choice alone), from the
    groups_kept best of n_groups equal runs of experts (a group counts as its best expert, or as
    the sum of its two best: group_score "max" / "top2"); ties go to the lowest expert. Weights
    are the scores, over their sum if renormalize, times scale. Experts at -inf or NaN are
    never chosen; a slot left over has id -1 and weight 0. Returns ((n, top_k) int32, (n, top_k) float32).
    """
    _cuda(logits, "logits")
    _need(logits.dtype in SRC_IDS and logits.dim() == 2, "logits must be a 2-D float32 / float16 / bfloat16 tensor")
    _need(score in _SCORES, f"score {score!r} is not one of {list(_SCORES)}")
    _need(group_score in _GROUP_SCORES, f"group_score {group_score!r} is not one of {list(_GROUP_SCORES)}")
    n, e = logits.shape
    if e and (logits.stride(1) != 1 or (n > 1 and logits.stride(0) < e)):
        logits = logits.contiguous()
    if bias is not None:
        _cuda(bias, "bias", logits.device)
        _need(bias.dtype == torch.float32 and bias.dim() == 1 and bias.shape[0] == e, f"bias must be {e} float32 values")
        bias = bias.contiguous()
    top_k = int(top_k)
    ids = torch.empty((n, max(top_k, 0)), dtype=torch.int32, device=logits.device)
    weights = torch.empty((n, max(top_k, 0)), dtype=torch.float32, device=logits.device)
    with torch.cuda.device(logits.device):
        check(lib().qs_route(logits.data_ptr(), SRC_IDS[logits.dtype], _row_stride(logits), n, e, top_k, _SCORES[score],
                             None if bias is None else bias.data_ptr(), int(n_groups), int(groups_kept),
                             _GROUP_SCORES[group_score], int(bool(renormalize)), float(scale), ids.data_ptr(),
                             weights.data_ptr(), _stream(logits.device)))
    return ids, weights


@dataclass(frozen=True)
class ExpertPlan:
    """Slots grouped by expert (expert_plan): what matmul_experts needs of a routing."""

    ids: torch.Tensor      # (tokens, top_k) int32
    order: torch.Tensor    # (tokens * top_k,) int32: slots by expert, those without one last
    offsets: torch.Tensor  # (experts + 1,) int32: where each expert's slots start
    n_experts: int


def expert_plan(ids: torch.Tensor, n_experts: int) -> ExpertPlan:
    """Group the slots of ids (tokens, top_k) int32 by expert; ids outside [0, n_experts) are
    slots without an expert. The plan keeps ids: do not change them while it is in use."""
    _cuda(ids, "ids")
    _need(ids.dtype == torch.int32 and ids.dim() == 2, "ids must be a (tokens, top_k) int32 tensor")
    ids = ids.contiguous()
    order = torch.empty(ids.numel(), dtype=torch.int32, device=ids.device)
    offsets = torch.empty(max(int(n_experts), 0) + 1, dtype=torch.int32, device=ids.device)
    with torch.cuda.device(ids.device):
        check(lib().qs_expert_plan(ids.data_ptr(), ids.numel(), int(n_experts), order.data_ptr(), offsets.data_ptr(), _stream(ids.device)))
    return ExpertPlan(ids, order, offsets, int(n_experts))


def _packed_args(blocks: torch.Tensor, ggml_type: int, x_q8: torch.Tensor, dims: int, out_dtype: torch.dtype) -> int:
    """Checks shared by the products; the row length k."""
    _cuda(blocks, "blocks")
    _need(blocks.dtype == torch.uint8 and blocks.dim() == dims and blocks.stride(-1) == 1,
          f"blocks must be a {dims}-D uint8 tensor with packed rows in its last dimension")
    qk, nb = block_info(ggml_type)
    _need(blocks.shape[-1] > 0 and blocks.shape[-1] % nb == 0, f"row of {blocks.shape[-1]} bytes is not a whole number of {nb}-byte blocks")
    k = blocks.shape[-1] // nb * qk
    _cuda(x_q8, "x_q8", blocks.device)
    _need(x_q8.dtype == torch.uint8 and x_q8.dim() == 2 and x_q8.stride(1) == 1 and x_q8.shape[1] == k // 32 * 34,
          f"x_q8 must be row-major (rows, {k // 32 * 34}) uint8 Q8_0 blocks, as many values as the weight rows have")
    _need(out_dtype in SRC_IDS, f"unsupported output dtype {out_dtype}")
    _need(min(blocks.shape) > 0, "no weights")
    return k


def _workspace(size: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def matmul(blocks: torch.Tensor, ggml_type: int, x_q8: torch.Tensor, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """(rows, n) products of packed weights (n, row bytes) with Q8_0 activations (rows, k / 32 * 34):
    the decoded activations times the decoded weights transposed. Level products are exact
    integers, scales and sums float32, rounded once to out_dtype. Row strides may exceed the rows;
    weight rows must start on multiples of 16 bytes for Q4_K / Q5_K, 8 for Q5_1 / IQ4_XS, 4 for
    Q4_1 / Q2_K, 2 for the others.
    """
    k = _packed_args(blocks, ggml_type, x_q8, 2, out_dtype)
    n, rows = blocks.shape[0], x_q8.shape[0]
    L = lib()
    size = ctypes.c_int64()
    check(L.qs_matmul_workspace(int(ggml_type), n, k, rows, ctypes.byref(size)))
    out = torch.empty((rows, n), dtype=out_dtype, device=blocks.device)
    ws = _workspace(size.value, blocks.device)
    with torch.cuda.device(blocks.device):
        check(L.qs_matmul(int(ggml_type), blocks.data_ptr(), _row_stride(blocks), n, k, x_q8.data_ptr(), _row_stride(x_q8), rows,
                          out.data_ptr(), SRC_IDS[out_dtype], n, None if ws is None else ws.data_ptr(), size.value, _stream(blocks.device)))
    return out


def matmul_experts(blocks: torch.Tensor, ggml_type: int, x_q8: torch.Tensor, plan: ExpertPlan,
                   weights: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Products of each token with the packed weights (experts, n, row bytes) of its experts.

    x_q8: one Q8_0 row per token, or per slot (token * top_k + j). Without weights: (tokens, top_k, n),
    zeros where a slot has no expert. With weights (tokens, top_k) float32: (tokens, n), the sum of
    weight * product over a token's slots that have an expert. Otherwise as matmul.
    """
    k = _packed_args(blocks, ggml_type, x_q8, 3, out_dtype)
    experts, n = blocks.shape[0], blocks.shape[1]
    _need(experts == plan.n_experts, f"the plan is for {plan.n_experts} experts, the weights have {experts}")
    tokens, top_k = plan.ids.shape
    _cuda(plan.ids, "the plan", blocks.device)
    per_slot = x_q8.shape[0] != tokens
    _need(x_q8.shape[0] in (tokens, tokens * top_k), f"x_q8 must have {tokens} or {tokens * top_k} rows")
    if weights is not None:
        _cuda(weights, "weights", blocks.device)
        _need(weights.dtype == torch.float32 and weights.shape == plan.ids.shape, "weights must be (tokens, top_k) float32")
        weights = weights.contiguous()
    shape = (tokens, top_k, n) if weights is None else (tokens, n)
    if tokens == 0 or top_k == 0:
        return torch.zeros(shape, dtype=out_dtype, device=blocks.device)
    row = blocks.stride(1) if n > 1 else max(blocks.stride(1), blocks.shape[2])
    expert = blocks.stride(0) if experts > 1 else max(blocks.stride(0), n * row)
    L = lib()
    size = ctypes.c_int64()
    check(L.qs_matmul_experts_workspace(int(ggml_type), experts, n, k, tokens, top_k, int(per_slot), int(weights is not None), ctypes.byref(size)))
    out = torch.empty(shape, dtype=out_dtype, device=blocks.device)
    ws = _workspace(size.value, blocks.device)
    with torch.cuda.device(blocks.device):
        check(L.qs_matmul_experts(int(ggml_type), blocks.data_ptr(), row, expert, experts, n, k, x_q8.data_ptr(), _row_stride(x_q8),
                                  int(per_slot), plan.ids.data_ptr(), plan.order.data_ptr(), plan.offsets.data_ptr(), tokens, top_k,
                                  None if weights is None else weights.data_ptr(), out.data_ptr(), SRC_IDS[out_dtype], n,
                                  None if ws is None else ws.data_ptr(), size.value, _stream(blocks.device)))
    return out
