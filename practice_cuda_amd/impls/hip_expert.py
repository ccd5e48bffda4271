"""Tokens sorted by expert and back, and the experts' int8 products between.

A layer of experts sends each token to a few of them. With ids [T, k], the
experts of each token, pair p = t * k + j is token t's j-th choice:

* ``hip_expert_sort``      pairs in the order of their experts (an ExpertPlan);
* ``hip_expert_dispatch``  the tokens' rows in that order, [T * k, H];
* ``hip_expert_bmm``       each expert's rows times its own int8 weights;
* ``hip_expert_combine``   the rows back at their tokens, weighted and summed.

Dispatch and combine have gradients. Nothing reads sizes back to the host, so
all of them can be captured into a graph. Kernels: csrc/expert_route.hip,
csrc/int8_bmm*.hip. The reference has batched products of equal matrices only
(fp8_training/fp8_bench/impls/triton_per_channel.py:271-427).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ..registry import QuantResult
from . import _common as C
from .hip_int8 import _refused, check_codes
from .hip_per_channel import _validate_scale

MAX_EXPERTS = 1024
MAX_CHOICES = 128


@dataclass(frozen=True)
class ExpertPlan:
    """Pairs in the order of their experts; int32, contiguous.

    order [T * k]: the pair at each place, those of an expert in their own order;
    place [T, k]: the place of each pair; starts [experts + 1]: the first place
    of each expert, and the end of the last. Pairs without an expert come last
    in order and have place -1 - place."""

    order: torch.Tensor
    place: torch.Tensor
    starts: torch.Tensor

    @property
    def experts(self) -> int:
        return self.starts.shape[0] - 1


def _is_index(t: torch.Tensor, ndim: int, device: torch.device) -> bool:
    return t.ndim == ndim and t.dtype == torch.int32 and t.device == device and t.is_contiguous()


def hip_expert_sort(ids: torch.Tensor, experts: int) -> ExpertPlan:
    """The plan of ids [T, k], int32 or int64, contiguous: the experts of each token.

    The sort is stable. An id that is negative or not below ``experts`` (a padded
    token, another rank's expert) stands for none: dispatch leaves zeros at such
    a pair's place, and combine leaves it out. Up to 1024 experts and 128
    choices. ids of a token may repeat."""
    if ids.ndim != 2 or ids.dtype not in (torch.int32, torch.int64) or not ids.is_contiguous():
        raise ValueError(f"ids must be contiguous int32 or int64 [T, k], got {ids.dtype}, {tuple(ids.shape)}, "
                         f"strides={ids.stride()}")
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"experts must be from 1 to {MAX_EXPERTS}, got {experts}")
    if ids.shape[1] > MAX_CHOICES:
        raise ValueError(f"at most {MAX_CHOICES} choices a token, got {ids.shape[1]}")
    if not ids.is_cuda:
        _lib.require_gpu_tensor(ids, "ids")
    pairs, device = ids.numel(), ids.device
    L = _lib.lib()
    need = L.pcamd_expert_sort_workspace(pairs, experts)
    if need < 0:
        _refused(need, "pcamd_expert_sort_workspace")
    order = torch.empty(pairs, dtype=torch.int32, device=device)
    place = torch.empty(ids.shape, dtype=torch.int32, device=device)
    starts = torch.empty(experts + 1, dtype=torch.int32, device=device)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    rc = _lib.launch(L.pcamd_expert_sort, ids, ids.data_ptr(), ids.element_size(), pairs, experts, order.data_ptr(),
                     place.data_ptr(), starts.data_ptr(), _lib.ptr(workspace), need)
    if rc != 0:
        _refused(rc, "pcamd_expert_sort")
    return ExpertPlan(order, place, starts)


def _check_rows(t: torch.Tensor, name: str, rows: int) -> None:
    if t.ndim != 2 or t.shape[0] != rows:
        raise ValueError(f"{name} must be [{rows}, width] for this plan, got {tuple(t.shape)}")
    if t.dtype not in C._INPUT_DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{name} must be contiguous along its last dimension; strides={t.stride()}")


def _check_place(plan: ExpertPlan, device: torch.device) -> None:
    if not _is_index(plan.place, 2, device) or plan.place.shape[1] > MAX_CHOICES:
        raise ValueError(f"the plan's place must be contiguous int32 [T, k <= {MAX_CHOICES}] on {device}, got "
                         f"{plan.place.dtype}, {tuple(plan.place.shape)} on {plan.place.device}")


def _dispatch(x: torch.Tensor, place: torch.Tensor) -> torch.Tensor:
    tokens, choices = place.shape
    width = x.shape[1]
    out = torch.empty((tokens * choices, width), dtype=x.dtype, device=x.device)
    rc = _lib.launch(_lib.lib().pcamd_expert_dispatch, x, x.data_ptr(), _lib.dtype_code(x.dtype), tokens, choices,
                     width, x.stride(0), place.data_ptr(), out.data_ptr(), width)
    if rc != 0:
        _refused(rc, "pcamd_expert_dispatch")
    return out


def _combine(rows: torch.Tensor, place: torch.Tensor, weights: Optional[torch.Tensor]) -> torch.Tensor:
    tokens, choices = place.shape
    width = rows.shape[1]
    out = torch.empty((tokens, width), dtype=rows.dtype, device=rows.device)
    rc = _lib.launch(_lib.lib().pcamd_expert_combine, rows, rows.data_ptr(), _lib.dtype_code(rows.dtype), tokens,
                     choices, width, rows.stride(0), place.data_ptr(), _lib.ptr(weights),
                     0 if weights is None else _lib.dtype_code(weights.dtype), out.data_ptr(), width)
    if rc != 0:
        _refused(rc, "pcamd_expert_combine")
    return out


def _rows_major(grad: torch.Tensor) -> torch.Tensor:
    return grad if grad.stride(1) == 1 or grad.shape[1] <= 1 else grad.contiguous()


def _tangent(t: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    """A tangent as a tensor that a kernel can read: of its input's type, rows contiguous, no lazy zeros or signs."""
    if t._is_zerotensor():
        return torch.zeros(like.shape, dtype=like.dtype, device=like.device)
    return _rows_major(t.resolve_neg().to(like.dtype))


class _Dispatch(torch.autograd.Function):
    """Linear, so a tangent is dispatched like its tokens; and with the forward-mode inputs off in jvp, the calls
    made there can be differentiated backward."""

    @staticmethod
    def forward(ctx, x, place):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(place)
        ctx.save_for_forward(place)
        return _dispatch(x, place)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return None, None
        C.refuse_tangents("expert_dispatch's gradient", grad)
        place, = ctx.saved_tensors
        return _combine(_rows_major(grad), place, None), None

    @staticmethod
    def jvp(ctx, x_t, _):
        place, = ctx.saved_tensors
        return _Dispatch.apply(_tangent(x_t, x_t), place)


class _Combine(torch.autograd.Function):
    """Linear in rows and in weights: the tangent is combine of the rows' with the weights, plus combine of the rows
    with the weights'. Each is rounded to the rows' type before they are added (and the sum once more): two calls of
    the one kernel, at up to three half steps."""

    @staticmethod
    def forward(ctx, rows, weights, place):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(rows, weights, place)
        ctx.save_for_forward(rows, weights, place)
        return _combine(rows, place, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return None, None, None
        rows, weights, place = ctx.saved_tensors
        C.refuse_tangents("expert_combine's gradient", grad, weights if ctx.needs_input_grad[0] else None,
                          rows if ctx.needs_input_grad[1] else None)
        grad = _rows_major(grad)
        tokens, choices = place.shape
        width = rows.shape[1]
        to_rows = to_weights = None
        if ctx.needs_input_grad[0]:
            to_rows = torch.empty((rows.shape[0], width), dtype=rows.dtype, device=rows.device)
        if ctx.needs_input_grad[1]:
            to_weights = torch.empty(weights.shape, dtype=torch.float32, device=rows.device)
        rc = _lib.launch(
            _lib.lib().pcamd_expert_combine_backward, rows,
            grad.data_ptr(), rows.data_ptr(), _lib.dtype_code(rows.dtype), tokens, choices, width, grad.stride(0),
            rows.stride(0), place.data_ptr(), weights.data_ptr(), _lib.dtype_code(weights.dtype),
            _lib.ptr(to_rows), width, _lib.ptr(to_weights))
        if rc != 0:
            _refused(rc, "pcamd_expert_combine_backward")
        if to_weights is not None and weights.dtype != torch.float32:
            to_weights = to_weights.to(weights.dtype)
        return to_rows, to_weights, None

    @staticmethod
    def jvp(ctx, rows_t, weights_t, _):
        rows, weights, place = ctx.saved_tensors
        parts = []
        if rows_t is not None:
            parts.append(_Combine.apply(_tangent(rows_t, rows), weights, place))
        if weights_t is not None:
            parts.append(_Combine.apply(rows, _tangent(weights_t, weights).contiguous(), place))
        return parts[0] if len(parts) == 1 else parts[0] + parts[1]


def hip_expert_dispatch(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """The rows of x [T, H] in the plan's order: [T * k, H], row s that of pair order[s].

    float32, bfloat16 or float16, contiguous along H, any row stride; places of
    pairs without an expert get zeros. The gradient of a token is the sum over
    its choices, in fp32, rounded once. A forward-mode tangent is dispatched as x
    is; the gradient itself has none."""
    _check_rows(x, "x", plan.place.shape[0])
    _check_place(plan, x.device)
    if not x.is_cuda:
        _lib.require_gpu_tensor(x, "x")
    if x.requires_grad and torch.is_grad_enabled() or C.has_tangent(x):
        return _Dispatch.apply(x, plan.place)
    return _dispatch(x, plan.place)


def hip_expert_combine(rows: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor) -> torch.Tensor:
    """Each token's rows, weighted and summed: out[t] = sum_j weights[t, j] rows[place[t, j]], [T, H].

    rows [T * k, H] in the plan's order: float32, bfloat16 or float16,
    contiguous along H, any row stride; weights [T, k], any of those types,
    contiguous. Sums are fp32, over the choices in their order, rounded once to
    the rows' type; pairs without an expert are left out. Gradients: of rows
    (zeros at places of pairs without an expert) and of weights (summed in fp32
    in a fixed order). Forward-mode tangents of both go through; the gradients
    themselves have none."""
    pairs, device = plan.place.numel(), rows.device
    _check_rows(rows, "rows", pairs)
    _check_place(plan, device)
    if (weights.shape != plan.place.shape or weights.dtype not in C._INPUT_DTYPES or weights.device != device
            or not weights.is_contiguous()):
        raise ValueError(f"weights must be contiguous float32, bfloat16 or float16 {tuple(plan.place.shape)} on "
                         f"{device}, got {weights.dtype}, {tuple(weights.shape)} on {weights.device}")
    if not rows.is_cuda:
        _lib.require_gpu_tensor(rows, "rows")
    if (rows.requires_grad or weights.requires_grad) and torch.is_grad_enabled() or C.has_tangent(rows, weights):
        return _Combine.apply(rows, weights, plan.place)
    return _combine(rows, plan.place, weights)


def hip_expert_bmm(
    a: QuantResult,
    b: QuantResult,
    plan: ExpertPlan,
    *,
    gather: bool = False,
    out_dtype: torch.dtype = torch.bfloat16,
    bias: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    activation: str = "none",
) -> torch.Tensor:
    """Rows in the plan's order times their experts' weights, int8 codes with scales.

    b: [experts, K, N] with scales per column (channel_axis=-1); a: with scales
    per row (-2), [T * k, K] in the plan's order, or with gather [T, K], the
    tokens, whose rows are found within the call (dispatch of 8-bit rows without
    writing them). Both as hip_int8_quant leaves them; bias: [experts, N], any
    strides; activations as hip_int8_bmm's. Returns [T * k, N] (N / 2 for
    "swiglu"): row s is that of pair order[s], and rows of pairs without an
    expert are zeros. There is no gradient: going backward is an error."""
    at, bt = a.tensor, b.tensor
    if at.ndim != 2 or bt.ndim != 3:
        raise ValueError(f"A must be [rows, K] and B [experts, K, N], got {tuple(at.shape)} and {tuple(bt.shape)}")
    act = check_codes(at, bt, out_dtype, activation)
    device = at.device
    _check_place(plan, device)
    tokens, choices = plan.place.shape
    pairs, experts = tokens * choices, bt.shape[0]
    if not (_is_index(plan.order, 1, device) and plan.order.shape[0] == pairs and _is_index(plan.starts, 1, device)
            and plan.starts.shape[0] == experts + 1):
        raise ValueError(f"the plan must be of {experts} experts and {pairs} pairs on {device}, got order "
                         f"{tuple(plan.order.shape)} and starts {tuple(plan.starts.shape)}")
    rows, k = at.shape
    if rows != (tokens if gather else pairs):
        raise ValueError(f"A must have {tokens if gather else pairs} rows with gather={gather}, got {rows}")
    cols = bt.shape[2]
    n = cols // 2 if activation == "swiglu" else cols
    _validate_scale(a, expected_shape=(rows,), expected_axis=-2, operand="A")
    _validate_scale(b, expected_shape=(experts, cols), expected_axis=-1, operand="B")
    if bias is not None and (bias.shape != (experts, cols) or bias.dtype not in C._INPUT_DTYPES
                             or bias.device != device):
        raise ValueError(f"bias must be float32, bfloat16 or float16 {(experts, cols)} on {device}, got {bias.dtype}, "
                         f"{tuple(bias.shape)} on {bias.device}")
    sa, sb = a.dequant_scale, b.dequant_scale
    record = ((sa.requires_grad or sb.requires_grad or bias is not None and bias.requires_grad)
              and torch.is_grad_enabled())
    C.refuse_tangents("expert_bmm", sa, sb, bias)
    if out is not None:
        if out.shape != (pairs, n) or out.dtype != out_dtype or out.device != device:
            raise ValueError(f"out must be {out_dtype} with shape {(pairs, n)} on {device}, got {out.dtype}, "
                             f"{tuple(out.shape)}, {out.device}")
        if out.stride(1) != 1 and n > 1:
            raise ValueError(f"out must be contiguous along its last dimension; strides={out.stride()}")
        if record:
            C.refuse_recorded("expert_bmm", "out")
    _lib.require_gpu_tensor(at, "A")
    if out is None:
        out = torch.empty((pairs, n), dtype=out_dtype, device=device)
    s_b, s_sb = bt.stride(), sb.stride()
    s_bias = (0, 0) if bias is None else bias.stride()
    rc = _lib.launch(
        _lib.lib().pcamd_expert_bmm_int8, at,
        at.data_ptr(), rows, bt.data_ptr(), experts, n, k, at.stride(0), s_b[0], s_b[2],
        out.data_ptr(), _lib.dtype_code(out_dtype), out.stride(0),
        _lib.ptr(bias), 0 if bias is None else _lib.dtype_code(bias.dtype), s_bias[0], s_bias[1],
        sa.data_ptr(), sa.stride(0), sb.data_ptr(), s_sb[0], s_sb[1],
        plan.starts.data_ptr(), plan.order.data_ptr() if gather else 0, pairs, choices, act)
    if rc != 0:
        _refused(rc, "pcamd_expert_bmm_int8")
    if record:
        out, = C.without_gradient("expert_bmm", (sa, sb, bias), out)
    return out
