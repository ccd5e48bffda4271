"""Int8 codes with one scale for each row, and the products of such codes.

``hip_int8_quant`` is the integer counterpart of ``hip_per_channel_quant``:

    top = max(max|x|, eps) over a row, scale = top / 127,
    code = rint(127 x / top), ties to even, of the real quotient

and ``hip_int8_bmm`` that of ``hip_per_channel_bmm``: the sums of products are
whole numbers, exact in 32 bits, and are multiplied once by both scales. Kernels:
csrc/int8_quant.hip, csrc/int8_bmm*.hip. The reference's quantized products are
fp8 (fp8_training/fp8_bench/impls/triton_per_channel.py:90-427); these keep its
shapes, axes and layouts.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ..registry import QuantResult
from . import _common as C
from .hip_per_channel import _validate_scale

_OUT_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_ACTIVATIONS = {"none": _lib.ACT_NONE, "gelu": _lib.ACT_GELU, "swiglu": _lib.ACT_SWIGLU}
MAX_K = 131071  # 128 * 128 * MAX_K < 2 ** 31


def hip_int8_quant(x: torch.Tensor, *, channel_axis: int = -2, eps: float = 1e-12) -> QuantResult:
    """Int8 codes of x [M, N] or [B, M, N], float32 / bfloat16 / float16.

    channel_axis=-2: one scale per row, x contiguous along N (a product's left
    operand); -1: one per column, x contiguous along M (its right operand: a
    weight [.., N, K] passed as ``w.transpose(-1, -2)``). Rows (columns) may
    have any strides, and up to 2^31 - 16385 values. The codes lie as x does, each row (column) at
    a multiple of 16 bytes, so the result may be a view of padded memory; eps is
    the floor of a row's maximum. A row with a NaN or an infinity gets codes of
    zero and a scale of NaN, which makes its products NaN. There is no gradient:
    going backward is an error."""
    if x.ndim not in (2, 3):
        raise ValueError(f"int8 quant expects a 2D or 3D tensor, got {tuple(x.shape)}")
    if channel_axis not in (-1, -2):
        raise ValueError(f"channel_axis must be -1 or -2, got {channel_axis}")
    dtype, device, shape = x.dtype, x.device, x.shape
    if dtype not in C._INPUT_DTYPES:
        raise ValueError(f"int8 quant input dtype must be float32, bfloat16 or float16, got {dtype}")
    if not 0 <= eps < 3e38:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    rows = x if channel_axis == -2 else x.transpose(-1, -2)
    strides = rows.stride()
    m, n = rows.shape[-2:]
    if strides[-1] != 1 and n > 1:
        raise ValueError(f"x must be contiguous along the dimension that its scales are for all of (channel_axis="
                         f"{channel_axis}); shape={tuple(shape)}, strides={x.stride()}")
    C.refuse_tangents("int8_quant", x)
    if not x.is_cuda:
        _lib.require_gpu_tensor(x, "x")
    flat = len(shape) == 2
    batch = 1 if flat else shape[0]
    pitch = -(-n // 16) * 16
    codes = torch.empty((m, pitch) if flat else (batch, m, pitch), dtype=torch.int8, device=device)
    scale = torch.empty((m,) if flat else (batch, m), dtype=torch.float32, device=device)
    rc = _lib.launch(
        _lib.lib().pcamd_quant_int8, x,
        x.data_ptr(), _lib.dtype_code(dtype), batch, m, n, 0 if flat else strides[0], strides[-2],
        codes.data_ptr(), m * pitch, pitch, scale.data_ptr(), m, 1, eps)
    if rc != 0:
        _refused(rc, "pcamd_quant_int8")
    if pitch != n:
        codes = codes[..., :n]
    if channel_axis == -1:
        codes = codes.transpose(-1, -2)
    if x.requires_grad and torch.is_grad_enabled():
        codes, scale = C.without_gradient("int8_quant", (x,), codes, scale)
    return QuantResult(codes, scale, "hip_int8", "channel",
                       {"logical_shape": tuple(shape), "dtype": "torch.int8", "channel_axis": channel_axis})


def _refused(rc: int, what: str) -> None:
    """Bad alignment and sizes past the kernels' are the caller's values."""
    if rc in (_lib.ERR_INVALID, _lib.ERR_UNSUPPORTED):
        raise ValueError(_lib.lib().pcamd_last_error().decode())
    _lib.check(rc, what)


def check_codes(a: torch.Tensor, b: torch.Tensor, out_dtype: torch.dtype, activation: str) -> int:
    """The activation's code; types, devices and layouts of a product's operands ([.., M, K] and [.., K, N])."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise ValueError(f"A and B must be int8 tensors, got {a.dtype} and {b.dtype}")
    if a.device != b.device:
        raise ValueError(f"A and B must be on the same device: A={a.device}, B={b.device}")
    k = a.shape[-1]
    if k != b.shape[-2]:
        raise ValueError(f"shape mismatch: A={tuple(a.shape)}, B={tuple(b.shape)}")
    if k > MAX_K:
        raise ValueError(f"K must be at most {MAX_K} (sums of 32 bits), got {k}")
    if k > 1 and (a.stride(-1) != 1 or b.stride(-2) != 1):
        raise ValueError(f"A and B must be contiguous along K; strides={a.stride()} and {b.stride()}")
    if activation == "swiglu" and b.shape[-1] % 2:
        raise ValueError(f"swiglu takes gates and others in halves of B's columns, got {b.shape[-1]}")
    if out_dtype not in _OUT_DTYPES:
        raise ValueError(f"unsupported out_dtype for the int8 product: {out_dtype}")
    return _ACTIVATIONS[activation]


def hip_int8_bmm(
    a: QuantResult,
    b: QuantResult,
    *,
    out_dtype: torch.dtype = torch.bfloat16,
    bias: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    activation: str = "none",
) -> torch.Tensor:
    """act((A @ B) * sa[b, m] * sb[b, n] + bias) of int8 codes.

    a: [B, M, K] with scales per row (channel_axis=-2), b: [B, K, N] with scales
    per column (-1), both contiguous along K, rows (columns) at multiples of 16
    bytes, as hip_int8_quant leaves them; K up to 131071, where the sums are
    exact, and B up to 65535. bias: [B, M, N], any strides. activation: "none", "gelu", or "swiglu",
    which takes the first half of b's columns as gates of the second: silu(gate)
    * other, [B, M, N / 2] (bias still has N columns). There is no gradient: going
    backward is an error."""
    at, bt = a.tensor, b.tensor
    if at.ndim != 3 or bt.ndim != 3:
        raise ValueError("BMM expects 3D quantized tensors")
    act = check_codes(at, bt, out_dtype, activation)
    batch, m, k = at.shape
    if bt.shape[0] != batch:
        raise ValueError(f"shape mismatch: A={tuple(at.shape)}, B={tuple(bt.shape)}")
    cols = bt.shape[2]
    n = cols // 2 if activation == "swiglu" else cols
    _validate_scale(a, expected_shape=(batch, m), expected_axis=-2, operand="A")
    _validate_scale(b, expected_shape=(batch, cols), expected_axis=-1, operand="B")
    given = out is not None
    if given or at.is_cuda:
        out = C.prepare_out(out, out_dtype, batch, m, n, at.device)
    bias, bias_strides, bias_code = C.check_bias(bias, batch, m, cols, at.device, require_n_contiguous=False)
    sa, sb = a.dequant_scale, b.dequant_scale
    C.refuse_tangents("int8_bmm", sa, sb, bias)
    _lib.require_gpu_tensor(at, "A")
    # the scales of a quantized input stand for it: its codes are whole numbers, which require no gradient
    record = ((sa.requires_grad or sb.requires_grad or bias is not None and bias.requires_grad)
              and torch.is_grad_enabled())
    if record and given:
        C.refuse_recorded("int8_bmm", "out")
    s_a, s_b, s_c, s_sa, s_sb = at.stride(), bt.stride(), out.stride(), sa.stride(), sb.stride()
    rc = _lib.launch(
        _lib.lib().pcamd_bmm_int8, at,
        at.data_ptr(), bt.data_ptr(), batch, m, n, k, s_a[0], s_a[1], s_b[0], s_b[2],
        out.data_ptr(), _lib.dtype_code(out_dtype), s_c[0], s_c[1], _lib.ptr(bias), bias_code, *bias_strides,
        sa.data_ptr(), s_sa[0], s_sa[1], sb.data_ptr(), s_sb[0], s_sb[1], act)
    if rc != 0:
        _refused(rc, "pcamd_bmm_int8")
    if record:
        out, = C.without_gradient("int8_bmm", (sa, sb, bias), out)
    return out
