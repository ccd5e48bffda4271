"""Root-mean-square norm with the residual's addition and an fp8 output.

``hip_rms_norm_quant(x, weight, residual=r)`` is, in one kernel,

    total = x + r                                   (fp32)
    y = total * rsqrt(mean(total ** 2) + norm_eps) * weight
    hip_per_block_quant(y, block_m=1, block_n=128)

with y in fp32 throughout (it is rounded once, to fp8), and returns the
QuantResult, the left operand of the block-scaled BMM, beside ``total`` rounded
to x's dtype, the next residual. The kernel is csrc/rms_norm.hip. The
reference has no counterpart: its layers quantize an activation that a norm
left in 16 bits (fp8_training/fp8_bench/impls/triton_per_block.py:60-150).
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ..registry import QuantResult
from . import _common as C

_GROUP = 128


_NAMES = {t: str(t) for t in C._FP8_DTYPES}


def hip_rms_norm_quant(
    x: torch.Tensor,
    weight: torch.Tensor,
    *,
    residual: Optional[torch.Tensor] = None,
    norm_eps: float = 1e-6,
    fp8_dtype: torch.dtype = torch.float8_e4m3fn,
    eps: float = 1e-12,
    residual_out: Optional[torch.Tensor] = None,
) -> tuple[QuantResult, Optional[torch.Tensor]]:
    """(fp8 of the normed rows with one scale per 1 x 128 group, x + residual).

    x: [M, N] or [B, M, N], float32 / bfloat16 / float16, contiguous along N
    (any row strides, any N); weight: [N], any of those dtypes; residual: as x.
    residual_out: where x + residual goes (a new tensor if None; it may be
    ``residual`` or ``x`` itself); None comes back where there is no residual.
    norm_eps is added to the mean square, eps is the amax floor of the
    quantization. A group with a NaN keeps it as a NaN code; its scale is that
    of the other values. There is no gradient: going backward is an error."""
    C.check_quant_input(x, fp8_dtype, "rms norm quant")
    shape, strides, dtype, device = x.shape, x.stride(), x.dtype, x.device
    n = shape[-1]
    if weight.shape != (n,) or n > 1 and weight.stride(0) != 1:
        raise ValueError(f"weight must be contiguous with shape ({n},), got {tuple(weight.shape)}, "
                         f"strides={weight.stride()}")
    if weight.dtype not in C._INPUT_DTYPES:
        raise ValueError(f"weight dtype must be float32, bfloat16 or float16, got {weight.dtype}")
    if strides[-1] != 1 and n > 1:
        raise ValueError(f"x must be contiguous along its last dimension; strides={strides}")
    if eps < 0 or norm_eps < 0:
        raise ValueError(f"eps and norm_eps must not be negative, got {eps} and {norm_eps}")
    if weight.device != device:
        raise ValueError(f"weight must be on {device}, got {weight.device}")
    flat = len(shape) == 2  # rows without a batch dimension: batch stride 0
    batch, m = (1, shape[0]) if flat else shape[:2]
    given = residual_out is not None
    if residual is None:
        if given:
            raise ValueError("residual_out needs a residual")
        residual_args, out_args = (0, 0, 0), (0, 0, 0)
    else:
        if not given:
            residual_out = torch.empty(shape, dtype=dtype, device=device)
        residual_args = _like(residual, "residual", shape, dtype, device, flat)
        out_args = _like(residual_out, "residual_out", shape, dtype, device, flat)
    C.refuse_tangents("rms_norm_quant", x, weight, residual)
    if not x.is_cuda:
        _lib.require_gpu_tensor(x, "x")
    record = ((x.requires_grad or weight.requires_grad or residual is not None and residual.requires_grad)
              and torch.is_grad_enabled())
    if record and given:
        C.refuse_recorded("rms_norm_quant", "residual_out")
    groups = -(-n // _GROUP)
    q = torch.empty(shape, dtype=fp8_dtype, device=device)
    scale = torch.empty((m, groups) if flat else (batch, m, groups), dtype=torch.float32, device=device)
    rc = _lib.launch(
        _lib.lib().pcamd_rms_norm_quant, x,
        x.data_ptr(), _lib.dtype_code(dtype), batch, m, n, 0 if flat else strides[0], strides[-2],
        *residual_args, weight.data_ptr(), _lib.dtype_code(weight.dtype),
        q.data_ptr(), _lib.dtype_code(fp8_dtype), m * n, n, scale.data_ptr(), m * groups, groups,
        *out_args, norm_eps, _lib.FP8_MAX[fp8_dtype], eps)
    _lib.check(rc, "pcamd_rms_norm_quant")
    if record:
        q, scale, residual_out = C.without_gradient("rms_norm_quant", (x, weight, residual), q, scale, residual_out)
    return QuantResult(q, scale, "hip_rms_norm", "block",
                       {"logical_shape": tuple(shape), "fp8_dtype": _NAMES[fp8_dtype], "block_m": 1,
                        "block_n": _GROUP}), residual_out


def _like(t: torch.Tensor, name: str, shape, dtype, device, flat: bool) -> tuple[int, int, int]:
    """(address, batch stride, row stride) of a tensor that has to be like x."""
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be like x ({tuple(shape)}, {dtype}, {device}), got "
                         f"{tuple(t.shape)}, {t.dtype}, {t.device}")
    strides = t.stride()
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous along its last dimension; strides={strides}")
    return t.data_ptr(), 0 if flat else strides[0], strides[-2]
