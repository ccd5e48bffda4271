"""Attention over one latent vector a token: its paged cache, the absorbed form
for decoding and the expanded form for prompts.

A layer of this kind keeps, for each token, a latent vector c (from which every
head's key and value are a linear map) and one rotary key that the heads share.
Two forms of the same attention follow:

* expanded (prompts): each head's keys W_k c and values W_v c are computed, and
  ``hip_latent_prefill`` attends over them;
* absorbed (decoding): q . (W_k c) = (W_k^T q) . c, so the query moves into the
  latent space (the head-batched product of the block-scaled BMM),
  ``hip_latent_decode`` attends over the cache itself, and W_v is applied to
  its output.

``hip_latent_append`` norms new tokens' latents and writes them into the cache.
Kernels: csrc/rms_norm.hip, csrc/latent_decode.h, csrc/latent_prefill.hip. The
reference has the products around these operators (its BMM's head-batched
shapes, kernels/fp8_bmm), not the operators.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Union

import torch

from .. import _lib
from . import _common as C

_TOKEN_DTYPES = (torch.bfloat16, torch.float16)
# (latent, rotary) widths of the decode kernels; (key, rotary, value) of the prefill kernels
DECODE_WIDTHS = ((512, 64), (256, 32))
PREFILL_WIDTHS = ((128, 64, 128), (64, 32, 64))


@dataclass(frozen=True)
class LatentCache:
    """Pages of a latent cache.

    latent: [pages, page_size, latent], bfloat16 / float16, or float8_e4m3fn
    codes; rope: [pages, page_size, rotary], bfloat16 / float16 (the queries'
    dtype); scale: with fp8 codes, float32 [pages, page_size, latent / 128],
    the scale that multiplies each token's 128 codes (what per_block_quant with
    1 x 128 blocks returns). latent and rope may be views of one buffer; each
    is contiguous along its last dimension, with 16-byte aligned rows.
    """

    latent: torch.Tensor
    rope: torch.Tensor
    scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages: int, page_size: int, *, latent_dim: int = 512, rope_dim: int = 64,
              dtype: torch.dtype = torch.bfloat16, fp8: bool = False,
              device: Union[str, torch.device] = "cuda") -> "LatentCache":
        """Uninitialised pages: the tokens' dtype, or fp8 with scales."""
        if dtype not in _TOKEN_DTYPES:
            raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}")
        if fp8 and latent_dim % 128:
            raise ValueError(f"an fp8 cache's latent width must be a multiple of 128, got {latent_dim}")
        shape = (pages, page_size)
        return cls(
            torch.empty((*shape, latent_dim), dtype=torch.float8_e4m3fn if fp8 else dtype, device=device),
            torch.empty((*shape, rope_dim), dtype=dtype, device=device),
            torch.empty((*shape, latent_dim // 128), dtype=torch.float32, device=device) if fp8 else None)


def _check_cache(cache: LatentCache, dtype: torch.dtype, device: torch.device):
    """(latent width, rotary width, pages, page size, arguments) of a well-formed cache; the
    arguments are its addresses, dtype and strides in the entry points' order."""
    latent, rope, scale = cache.latent, cache.rope, cache.scale
    shape, sl, sr = latent.shape, latent.stride(), rope.stride()
    if len(shape) != 3 or rope.ndim != 3 or shape[:2] != rope.shape[:2]:
        raise ValueError("a cache's latent and rope must be [pages, page_size, width]; got "
                         f"{tuple(latent.shape)} and {tuple(rope.shape)}")
    pages, page, dl = shape
    kind = latent.dtype
    if page < 1:
        raise ValueError("a cache's pages must hold at least one token")
    if rope.dtype != dtype:
        raise ValueError(f"the cache's rope must have the tokens' dtype {dtype}, got {rope.dtype}")
    if sl[2] != 1 or sr[2] != 1:
        raise ValueError("a cache must be contiguous along its last dimension")
    if latent.device != device or rope.device != device:
        raise ValueError(f"the cache must be on {device}, got {latent.device} and {rope.device}")
    if kind == torch.float8_e4m3fn:
        if scale is None:
            raise ValueError("an fp8 cache needs its scales")
        if scale.shape != (pages, page, dl // 128) or scale.dtype != torch.float32 or scale.device != device:
            raise ValueError(f"the cache's scale must be float32 with shape {(pages, page, dl // 128)} on {device}, "
                             f"got {scale.dtype}, {tuple(scale.shape)}, {scale.device}")
        ss = scale.stride()
        if ss[2] != 1 and dl > 128:
            raise ValueError("the cache's scale must be contiguous along its last dimension")
        scale_args = (scale.data_ptr(), ss[0], ss[1])
    else:
        if kind != dtype:
            raise ValueError(f"the cache's latent must be {dtype} or float8_e4m3fn, got {kind}")
        if scale is not None:
            raise ValueError("only an fp8 cache has scales")
        scale_args = (0, 0, 0)
    return dl, rope.shape[2], pages, page, (latent.data_ptr(), _lib.dtype_code(kind), sl[0], sl[1],
                                            rope.data_ptr(), sr[0], sr[1], *scale_args, pages, page)


def hip_latent_append(
    cache: LatentCache,
    latent: torch.Tensor,
    rope: torch.Tensor,
    slots: torch.Tensor,
    *,
    weight: Optional[torch.Tensor] = None,
    norm_eps: float = 1e-6,
    eps: float = 1e-12,
) -> LatentCache:
    """Write new tokens into the cache; returns it.

    latent [T, latent] and rope [T, rotary], bfloat16 or float16, contiguous
    along their last dimension (views of one projection's output, say); slots:
    int32 or int64 [T], page * page_size + place. A token whose slot is
    negative or past the cache is left out. Slots that are read later must be
    distinct: tokens of one slot are written side by side, in no order, and may
    leave one's codes with another's scales or rotary key (a slot that padded
    tokens share may hold anything). weight: the root-mean-square norm's, applied to the latents in fp32
    first (None: no norm). An fp8 cache gets hip_per_block_quant's codes and
    scales of 1 x 128 groups, with eps as the amax floor."""
    if latent.ndim != 2 or rope.ndim != 2 or latent.shape[0] != rope.shape[0]:
        raise ValueError(f"latent and rope must be [T, width], got {tuple(latent.shape)} and {tuple(rope.shape)}")
    dtype, device = latent.dtype, latent.device
    if dtype not in _TOKEN_DTYPES or rope.dtype != dtype:
        raise ValueError(f"latent and rope must both be bfloat16 or float16, got {dtype} and {rope.dtype}")
    tokens = latent.shape[0]
    sl, sr = latent.stride(), rope.stride()
    if sl[1] != 1 or sr[1] != 1:
        raise ValueError("latent and rope must be contiguous along their last dimension")
    if slots.shape != (tokens,) or slots.dtype not in (torch.int32, torch.int64) or tokens > 1 and slots.stride(0) != 1:
        raise ValueError(f"slots must be contiguous int32 or int64 with shape ({tokens},), got {slots.dtype}, "
                         f"{tuple(slots.shape)}")
    if slots.device != device or rope.device != device:
        raise ValueError(f"slots and rope must be on {device}, got {slots.device} and {rope.device}")
    dl, dr, _, _, cache_args = _check_cache(cache, dtype, device)
    if latent.shape[1] != dl or rope.shape[1] != dr:
        raise ValueError(f"the cache holds widths {dl} and {dr}, got {latent.shape[1]} and {rope.shape[1]}")
    if weight is not None:
        if weight.shape != (dl,) or weight.stride(0) != 1 or weight.dtype not in C._INPUT_DTYPES:
            raise ValueError(f"weight must be contiguous float32, bfloat16 or float16 with shape ({dl},), got "
                             f"{weight.dtype}, {tuple(weight.shape)}")
        if weight.device != device:
            raise ValueError(f"weight must be on {device}, got {weight.device}")
    if eps < 0 or norm_eps < 0:
        raise ValueError(f"eps and norm_eps must not be negative, got {eps} and {norm_eps}")
    if not latent.is_cuda:
        _lib.require_gpu_tensor(latent, "latent")
    if ((latent.requires_grad or rope.requires_grad or weight is not None and weight.requires_grad)
            and torch.is_grad_enabled()):
        C.refuse_recorded("latent_append", "the cache")
    rc = _lib.launch(
        _lib.lib().pcamd_latent_append, latent,
        latent.data_ptr(), rope.data_ptr(), _lib.dtype_code(dtype), tokens, dl, dr, sl[0], sr[0],
        _lib.ptr(weight), 0 if weight is None else _lib.dtype_code(weight.dtype), slots.data_ptr(), slots.element_size(), *cache_args, norm_eps, eps)
    if rc == _lib.ERR_UNSUPPORTED:
        raise ValueError(_lib.lib().pcamd_last_error().decode())
    _lib.check(rc, "pcamd_latent_append")
    return cache


def _check_out(out: Optional[torch.Tensor], shape: tuple, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    if tuple(out.shape) != shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"out must be {like.dtype} with shape {shape} on {like.device}, got {out.dtype}, "
                         f"{tuple(out.shape)}, {out.device}")
    if out.stride(-1) != 1:
        raise ValueError(f"out must be contiguous along its last dimension; strides={out.stride()}")
    return out


def _check_aligned(rows) -> None:
    """Rows that the kernels read in 16-byte pieces (names with their tensors)."""
    for name, t in rows:
        size = t.element_size()
        if t.data_ptr() % 16 or any(s * size % 16 for s, n in zip(t.stride()[:-1], t.shape) if n > 1):
            raise ValueError(f"{name} must have 16-byte aligned rows; strides={t.stride()}, "
                             f"address % 16 = {t.data_ptr() % 16}")


def hip_latent_decode(
    q_latent: torch.Tensor,
    q_rope: torch.Tensor,
    cache: LatentCache,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    softmax_scale: float,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
):
    """Attention of S new tokens a sequence over the paged cache, absorbed form.

    q_latent [B, S, H, latent] and q_rope [B, S, H, rotary]: bfloat16 or
    float16, contiguous along the last dimension, any other strides (a
    head-batched product's [H, B * S, latent] viewed so, say). block_table:
    int32 [B, max_pages], the pages of each sequence in order; seq_lens: int32
    [B], its tokens, the S new ones (already in the cache) among them. New
    token i sees the tokens before seq_lens - S + i + 1; a row that sees none,
    as of a padded batch's empty sequence, gives zeros and a log-sum of -inf.
    Lengths past the table's pages are cut to them, and page numbers past the
    cache read one of its own pages. What lies behind a sequence's last token
    in its page is never used, whatever it holds; a NaN or infinity in a
    token reaches the rows that see it and may reach the same sequence's
    earlier new tokens, which do not.

    An fp8 cache's scales may have any size under bfloat16 queries, and up to
    2^15 under float16 ones, whose attention weights are multiplied by them.

    Returns out [B, S, H, latent] in the queries' dtype and, with return_lse,
    float32 [B, S, H]: the natural logarithm of the sum of exponentials. There
    is no gradient: going backward is an error."""
    if q_latent.ndim != 4 or q_rope.ndim != 4 or q_latent.shape[:3] != q_rope.shape[:3]:
        raise ValueError("queries must be [B, S, H, width], got "
                         f"{tuple(q_latent.shape)} and {tuple(q_rope.shape)}")
    dtype, device = q_latent.dtype, q_latent.device
    if dtype not in _TOKEN_DTYPES or q_rope.dtype != dtype:
        raise ValueError(f"queries must both be bfloat16 or float16, got {dtype} and {q_rope.dtype}")
    sl, sr = q_latent.stride(), q_rope.stride()
    if sl[3] != 1 or sr[3] != 1:
        raise ValueError("queries must be contiguous along their last dimension")
    if q_rope.device != device:
        raise ValueError(f"q_rope must be on {device}, got {q_rope.device}")
    batch, new, heads, width = q_latent.shape
    dl, dr, _, page, cache_args = _check_cache(cache, dtype, device)
    if (dl, dr) not in DECODE_WIDTHS:
        raise ValueError(f"latent and rotary widths must be one of {DECODE_WIDTHS}, got {(dl, dr)}")
    if width != dl or q_rope.shape[3] != dr:
        raise ValueError(f"the cache holds widths {dl} and {dr}, got queries of {width} and {q_rope.shape[3]}")
    if (block_table.ndim != 2 or block_table.shape[0] != batch or block_table.dtype != torch.int32
            or block_table.device != device or block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be int32 [{batch}, max_pages], contiguous along its rows, on {device}; "
                         f"got {block_table.dtype}, {tuple(block_table.shape)}, {block_table.device}")
    if (seq_lens.shape != (batch,) or seq_lens.dtype != torch.int32 or seq_lens.device != device
            or batch > 1 and seq_lens.stride(0) != 1):
        raise ValueError(f"seq_lens must be contiguous int32 with shape ({batch},) on {device}; "
                         f"got {seq_lens.dtype}, {tuple(seq_lens.shape)}, {seq_lens.device}")
    record = (q_latent.requires_grad or q_rope.requires_grad) and torch.is_grad_enabled()
    if record and out is not None:
        C.refuse_recorded("latent_decode", "out")
    out = _check_out(out, (batch, new, heads, dl), q_latent)
    rows = (("q_latent", q_latent), ("q_rope", q_rope), ("the cache's latent", cache.latent),
            ("the cache's rope", cache.rope), ("out", out))
    if not q_latent.is_cuda:
        _check_aligned(rows)
        _lib.require_gpu_tensor(q_latent, "q_latent")
    lse = torch.empty((batch, new, heads), dtype=torch.float32, device=device) if return_lse else None
    L = _lib.lib()
    max_pages = block_table.shape[1]
    need = L.pcamd_latent_decode_workspace(batch, new, heads, dl, page, max_pages)
    if need < 0:
        raise ValueError(L.pcamd_last_error().decode())
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    so = out.stride()
    rc = _lib.launch(
        L.pcamd_latent_decode, q_latent,
        q_latent.data_ptr(), q_rope.data_ptr(), _lib.dtype_code(dtype), batch, new, heads, dl, dr,
        sl[0], sl[1], sl[2], sr[0], sr[1], sr[2], *cache_args,
        block_table.data_ptr(), block_table.stride(0), max_pages, seq_lens.data_ptr(),
        out.data_ptr(), so[0], so[1], so[2], _lib.ptr(lse), new * heads, heads, 1,
        softmax_scale, _lib.ptr(workspace), need)
    if rc != 0:
        _refused(rc, "pcamd_latent_decode", rows)
    if record:
        out, lse = C.without_gradient("latent_decode", (q_latent, q_rope), out, lse)
    return (out, lse) if return_lse else out


def _refused(rc: int, what: str, rows) -> None:
    """What a launch did not take: bad alignment and sizes past the kernels' are the caller's values."""
    if rc == _lib.ERR_INVALID:
        _check_aligned(rows)
    if rc == _lib.ERR_UNSUPPORTED:
        raise ValueError(_lib.lib().pcamd_last_error().decode())
    _lib.check(rc, what)


def hip_latent_prefill(
    q: torch.Tensor,
    k_nope: torch.Tensor,
    k_rope: torch.Tensor,
    v: torch.Tensor,
    cu_q: torch.Tensor,
    cu_k: torch.Tensor,
    *,
    softmax_scale: Optional[float] = None,
    causal: bool = True,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
):
    """Attention of packed sequences, expanded form.

    q [Tq, H, key + rotary], k_nope [Tk, H, key], k_rope [Tk, rotary] (shared
    by the heads), v [Tk, H, value]: bfloat16 or float16, contiguous along the
    last dimension (k_nope and v may be views of one projection's output).
    cu_q, cu_k: int32 [n + 1], the sequences' first tokens and the end of the
    last one. causal: query i of a sequence with nq queries and nk keys sees
    its first nk - nq + i + 1 keys, so a chunk may follow keys of earlier
    chunks. Rows that see no key, and queries ahead of the first sequence or
    behind the last, give zeros and a log-sum of -inf. softmax_scale: default
    (key + rotary) ** -0.5. A NaN or infinity in a value reaches the queries
    that see it and may reach up to 31 earlier ones of its sequence.

    Returns out [Tq, H, value] in q's dtype and, with return_lse, float32
    [Tq, H]: the natural logarithm of the sum of exponentials. There is no
    gradient: going backward is an error."""
    if q.ndim != 3 or k_nope.ndim != 3 or k_rope.ndim != 2 or v.ndim != 3:
        raise ValueError("q, k_nope and v must be [T, H, width] and k_rope [T, width]; got "
                         f"{tuple(q.shape)}, {tuple(k_nope.shape)}, {tuple(v.shape)} and {tuple(k_rope.shape)}")
    total_q, heads, dk = q.shape
    total_k, _, dn = k_nope.shape
    dr, dv = k_rope.shape[1], v.shape[2]
    if k_nope.shape[1] != heads or v.shape[:2] != k_nope.shape[:2] or k_rope.shape[0] != total_k:
        raise ValueError(f"keys and values do not go together: q {tuple(q.shape)}, k_nope {tuple(k_nope.shape)}, "
                         f"k_rope {tuple(k_rope.shape)}, v {tuple(v.shape)}")
    if (dn, dr, dv) not in PREFILL_WIDTHS or dk != dn + dr:
        raise ValueError(f"key, rotary and value widths must be one of {PREFILL_WIDTHS} and q's their key and rotary "
                         f"widths together; got {(dn, dr, dv)} and {dk}")
    dtype, device = q.dtype, q.device
    if dtype not in _TOKEN_DTYPES:
        raise ValueError(f"q must be bfloat16 or float16, got {dtype}")
    for t, name in ((k_nope, "k_nope"), (k_rope, "k_rope"), (v, "v")):
        if t.dtype != dtype or t.device != device:
            raise ValueError(f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    sq, sk, sr, sv = q.stride(), k_nope.stride(), k_rope.stride(), v.stride()
    for strides, name in ((sq, "q"), (sk, "k_nope"), (sr, "k_rope"), (sv, "v")):
        if strides[-1] != 1:
            raise ValueError(f"{name} must be contiguous along its last dimension; strides={strides}")
    for t, name in ((cu_q, "cu_q"), (cu_k, "cu_k")):
        if (t.ndim != 1 or t.shape != cu_q.shape or t.shape[0] < 1 or t.dtype != torch.int32 or t.device != device
                or t.stride(0) != 1):
            raise ValueError(f"cu_q and cu_k must be contiguous int32 [n + 1] on {device}; {name} is {t.dtype}, "
                             f"{tuple(t.shape)}, {t.device}")
    record = ((q.requires_grad or k_nope.requires_grad or k_rope.requires_grad or v.requires_grad)
              and torch.is_grad_enabled())
    if record and out is not None:
        C.refuse_recorded("latent_prefill", "out")
    out = _check_out(out, (total_q, heads, dv), q)
    rows = (("q", q), ("k_nope", k_nope), ("k_rope", k_rope), ("v", v), ("out", out))
    if not q.is_cuda:
        _check_aligned(rows)
        _lib.require_gpu_tensor(q, "q")
    lse = torch.empty((total_q, heads), dtype=torch.float32, device=device) if return_lse else None
    so = out.stride()
    rc = _lib.launch(
        _lib.lib().pcamd_latent_prefill, q,
        q.data_ptr(), k_nope.data_ptr(), k_rope.data_ptr(), v.data_ptr(), _lib.dtype_code(dtype),
        total_q, total_k, heads, dn, dr, dv, sq[0], sq[1], sk[0], sk[1], sr[0], sv[0], sv[1],
        cu_q.data_ptr(), cu_k.data_ptr(), cu_q.shape[0] - 1, out.data_ptr(), so[0], so[1], _lib.ptr(lse), heads, 1,
        1.0 / math.sqrt(dk) if softmax_scale is None else softmax_scale, 1 if causal else 0)
    if rc != 0:
        _refused(rc, "pcamd_latent_prefill", rows)
    if record:
        out, lse = C.without_gradient("latent_prefill", (q, k_nope, k_rope, v), out, lse)
    return (out, lse) if return_lse else out
