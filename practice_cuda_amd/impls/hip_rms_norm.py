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


def _rows(t: torch.Tensor) -> tuple[int, int]:
    """(batch, row) strides of a 2D or 3D tensor."""
    return (0, t.stride(0)) if t.ndim == 2 else (t.stride(0), t.stride(1))


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
    of the other values."""
    C.check_quant_input(x, fp8_dtype, "rms norm quant")
    n = x.shape[-1]
    if weight.shape != (n,) or weight.stride(0) != 1 and n > 1:
        raise ValueError(f"weight must be contiguous with shape ({n},), got {tuple(weight.shape)}, "
                         f"strides={weight.stride()}")
    if weight.dtype not in C._INPUT_DTYPES:
        raise ValueError(f"weight dtype must be float32, bfloat16 or float16, got {weight.dtype}")
    if x.stride(-1) != 1 and n > 1:
        raise ValueError(f"x must be contiguous along its last dimension; strides={x.stride()}")
    if eps < 0 or norm_eps < 0:
        raise ValueError(f"eps and norm_eps must not be negative, got {eps} and {norm_eps}")
    if weight.device != x.device:
        raise ValueError(f"weight must be on {x.device}, got {weight.device}")
    if residual is None:
        if residual_out is not None:
            raise ValueError("residual_out needs a residual")
        srb = srm = sob = som = 0
    else:
        if residual_out is None:
            residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        for t, name in ((residual, "residual"), (residual_out, "residual_out")):
            if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
                raise ValueError(f"{name} must be like x ({tuple(x.shape)}, {x.dtype}, {x.device}), got "
                                 f"{tuple(t.shape)}, {t.dtype}, {t.device}")
            if t.stride(-1) != 1 and n > 1:
                raise ValueError(f"{name} must be contiguous along its last dimension; strides={t.stride()}")
        (srb, srm), (sob, som) = _rows(residual), _rows(residual_out)
    _lib.require_gpu_tensor(x, "x")
    groups = -(-n // _GROUP)
    q = torch.empty(x.shape, dtype=fp8_dtype, device=x.device)
    scale = torch.empty((*x.shape[:-1], groups), dtype=torch.float32, device=x.device)
    batch, m = (1, x.shape[0]) if x.ndim == 2 else (x.shape[0], x.shape[1])
    rc = _lib.launch(
        _lib.lib().pcamd_rms_norm_quant, x,
        x.data_ptr(), _lib.dtype_code(x.dtype), batch, m, n, *_rows(x),
        _lib.ptr(residual), srb, srm, weight.data_ptr(), _lib.dtype_code(weight.dtype),
        q.data_ptr(), _lib.dtype_code(fp8_dtype), m * n, n, scale.data_ptr(), m * groups, groups,
        _lib.ptr(residual_out), sob, som, float(norm_eps), _lib.FP8_MAX[fp8_dtype], float(eps))
    _lib.check(rc, "pcamd_rms_norm_quant")
    result = QuantResult(
        tensor=q, dequant_scale=scale, impl="hip_rms_norm", granularity="block",
        meta={"logical_shape": tuple(x.shape), "fp8_dtype": str(fp8_dtype), "block_m": 1, "block_n": _GROUP})
    return result, residual_out
