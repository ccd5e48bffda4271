"""What the norm and latent attention entry points refuse, on the CPU (no kernel
is launched on these paths)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd import _lib

BF16, FP16 = torch.bfloat16, torch.float16
FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first


def refuses(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


# ---------------------------------------------------------------------------
# rms_norm_quant
# ---------------------------------------------------------------------------
def test_norm_refusals():
    x, w = torch.zeros((4, 256), dtype=BF16), torch.ones(256, dtype=BF16)
    f = pca.rms_norm_quant
    refuses("2D or 3D", f, x[0], w)
    refuses("input dtype", f, x.double(), w)
    refuses("fp8_dtype", f, x, w, fp8_dtype=torch.int8)
    refuses("weight must be contiguous", f, x, w[:128])
    refuses("weight must be contiguous", f, x[:, :128], w[::2])
    refuses("weight dtype", f, x, w.double())
    refuses("last dimension", f, x.t(), w[:4])
    refuses("not be negative", f, x, w, eps=-1.0)
    refuses("not be negative", f, x, w, norm_eps=-1.0)
    refuses("residual must be like x", f, x, w, residual=x.float())
    refuses("residual must be like x", f, x, w, residual=x[:3])
    refuses("residual_out must be like x", f, x, w, residual=x, residual_out=x[:3])
    refuses("residual must be contiguous", f, x[:, :4], w[:4], residual=torch.zeros((4, 4), dtype=BF16).t())
    refuses("needs a residual", f, x, w, residual_out=x)
    refuses("GPU tensor", f, x, w)


def test_norm_entry_refusals():
    L = _lib.lib()

    def call(x_dtype=_lib.BF16, m=4, n=256, res=None, w=FAKE, w_dtype=_lib.BF16, y_dtype=_lib.E4M3FN, out=None,
             norm_eps=1e-6, fp8_max=448.0, eps=1e-12):
        return L.pcamd_rms_norm_quant(FAKE, x_dtype, 1, m, n, 0, 256, res, 0, 256, w, w_dtype, FAKE, y_dtype, 0, 256,
                                      FAKE, 0, 2, out, 0, 256, norm_eps, fp8_max, eps, None)

    for kw, text in (({"x_dtype": 3}, b"x dtype"), ({"w_dtype": 9}, b"weight dtype"), ({"y_dtype": 1}, b"fp8 dtype"),
                     ({"m": -1}, b"negative"), ({"w": None}, b"null"), ({"res": FAKE}, b"come together"),
                     ({"out": FAKE}, b"come together"), ({"norm_eps": -1.0}, b"eps"), ({"fp8_max": 0.0}, b"fp8_max"),
                     ({"eps": float("nan")}, b"eps")):
        assert call(**kw) == _lib.ERR_INVALID, kw
        assert text in L.pcamd_last_error(), kw
    assert call(m=0) == _lib.OK and call(n=0) == _lib.OK


# ---------------------------------------------------------------------------
# the cache and append
# ---------------------------------------------------------------------------
def cpu_cache(**kw):
    return pca.LatentCache.empty(4, 16, device="cpu", **kw)


def test_cache():
    c = cpu_cache()
    assert c.latent.shape == (4, 16, 512) and c.rope.shape == (4, 16, 64) and c.scale is None
    c = cpu_cache(latent_dim=256, rope_dim=32, dtype=FP16, fp8=True)
    assert c.latent.dtype == torch.float8_e4m3fn and c.rope.dtype == FP16 and c.scale.shape == (4, 16, 2)
    refuses("dtype", cpu_cache, dtype=torch.float32)
    refuses("multiple of 128", cpu_cache, fp8=True, latent_dim=100)


def bad_caches():
    c, f = cpu_cache(), cpu_cache(fp8=True)
    yield "page_size, width", pca.LatentCache(c.latent, c.rope[:3])
    yield "page_size, width", pca.LatentCache(c.latent[0], c.rope[0])
    yield "at least one token", pca.LatentCache(c.latent[:, :0], c.rope[:, :0])
    yield "tokens' dtype", pca.LatentCache(c.latent, c.rope.half())
    yield "bfloat16 or float8_e4m3fn", pca.LatentCache(c.latent.half(), c.rope)
    yield "bfloat16 or float8_e4m3fn", pca.LatentCache(c.latent.to(torch.float8_e5m2), c.rope)
    yield "contiguous", pca.LatentCache(torch.zeros((4, 512, 16), dtype=BF16).transpose(1, 2), c.rope)
    yield "needs its scales", pca.LatentCache(f.latent, f.rope)
    yield "scale must be float32", pca.LatentCache(f.latent, f.rope, f.scale[..., :3])
    yield "scale must be float32", pca.LatentCache(f.latent, f.rope, f.scale.double())
    yield "scale must be contiguous", pca.LatentCache(f.latent, f.rope, torch.zeros((4, 4, 16)).transpose(1, 2))
    yield "only an fp8 cache", pca.LatentCache(c.latent, c.rope, f.scale)


def test_append_refusals():
    c = cpu_cache()
    latent, rope = torch.zeros((3, 512), dtype=BF16), torch.zeros((3, 64), dtype=BF16)
    slots = torch.arange(3)
    f = pca.latent_append
    for match, bad in bad_caches():
        refuses(match, f, bad, latent, rope, slots)
    refuses("T, width", f, c, latent, rope[:2], slots)
    refuses("T, width", f, c, latent[0], rope[0], slots)
    refuses("both be bfloat16 or float16", f, c, latent.float(), rope.float(), slots)
    refuses("both be bfloat16 or float16", f, c, latent, rope.half(), slots)
    refuses("last dimension", f, c, torch.zeros((512, 3), dtype=BF16).t(), rope, slots)
    refuses("slots", f, c, latent, rope, slots[:2])
    refuses("slots", f, c, latent, rope, slots.float())
    refuses("slots", f, c, latent, rope, torch.arange(6)[::2])
    refuses("widths", f, c, latent[:, :256], rope, slots)
    refuses("weight must be contiguous", f, c, latent, rope, slots, weight=torch.ones(256))
    refuses("weight must be contiguous", f, c, latent, rope, slots, weight=torch.ones(512).double())
    refuses("not be negative", f, c, latent, rope, slots, eps=-1.0)
    refuses("GPU tensor", f, c, latent, rope, slots)


def test_append_entry_refusals():
    L = _lib.lib()

    def call(dtype=_lib.BF16, dl=512, dr=64, cache_dtype=_lib.BF16, slot_bytes=8, page=16, pages=4, slots=FAKE,
             scale=None, tokens=3):
        return L.pcamd_latent_append(FAKE, FAKE, dtype, tokens, dl, dr, 576, 576, None, 0, slots, slot_bytes, FAKE,
                                     cache_dtype, 8192, 512, FAKE, 1024, 64, scale, 64, 4, pages, page, 1e-6, 1e-12,
                                     None)

    for kw, code, text in (({"dtype": _lib.F32}, _lib.ERR_INVALID, b"bf16 or fp16"),
                           ({"cache_dtype": _lib.F16}, _lib.ERR_INVALID, b"cache holds"),
                           ({"dl": 192}, _lib.ERR_UNSUPPORTED, b"multiple of 128"),
                           ({"dl": 640}, _lib.ERR_UNSUPPORTED, b"multiple of 128"),
                           ({"dr": 12}, _lib.ERR_UNSUPPORTED, b"multiple of 8"),
                           ({"slot_bytes": 2}, _lib.ERR_INVALID, b"int32 or int64"),
                           ({"page": 0}, _lib.ERR_INVALID, b"page size"),
                           ({"slots": None}, _lib.ERR_INVALID, b"null"),
                           ({"cache_dtype": _lib.E4M3FN}, _lib.ERR_INVALID, b"null"),
                           ({"tokens": -1}, _lib.ERR_INVALID, b"negative"),
                           ({"pages": 2 ** 60}, _lib.ERR_INVALID, b"too many")):
        assert call(**kw) == code, kw
        assert text in L.pcamd_last_error(), kw
    assert call(tokens=0) == _lib.OK and call(pages=0) == _lib.OK


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def test_decode_refusals():
    c = cpu_cache()
    ql, qr = torch.zeros((2, 1, 16, 512), dtype=BF16), torch.zeros((2, 1, 16, 64), dtype=BF16)
    table, lens = torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32)

    def f(ql=ql, qr=qr, cache=c, table=table, lens=lens, **kw):
        return pca.latent_decode(ql, qr, cache, table, lens, softmax_scale=0.1, **kw)

    for match, bad in bad_caches():
        refuses(match, f, cache=bad)
    refuses("B, S, H, width", f, ql=ql[0], qr=qr[0])
    refuses("B, S, H, width", f, qr=qr[:1])
    refuses("both be bfloat16 or float16", f, ql=ql.float(), qr=qr.float())
    refuses("both be bfloat16 or float16", f, qr=qr.half())
    refuses("last dimension", f, ql=torch.zeros((2, 1, 512, 16), dtype=BF16).transpose(2, 3))
    refuses("latent and rotary widths", f, ql=ql[..., :128], qr=qr[..., :32],
            cache=cpu_cache(latent_dim=128, rope_dim=32))
    refuses("cache holds widths", f, ql=ql[..., :256])
    refuses("block_table", f, table=table[:1])
    refuses("block_table", f, table=table.long())
    refuses("block_table", f, table=torch.zeros((3, 2), dtype=torch.int32).t())
    refuses("seq_lens", f, lens=lens[:1])
    refuses("seq_lens", f, lens=lens.long())
    refuses("out must be", f, out=ql[:1])
    refuses("out must be", f, out=ql.half())
    refuses("out must be contiguous", f, out=torch.zeros((2, 1, 512, 16), dtype=BF16).transpose(2, 3))
    odd = torch.zeros((2, 1, 16, 516), dtype=BF16)
    refuses("q_latent must have 16-byte aligned rows", f, ql=odd[..., :512])
    refuses("q_latent must have 16-byte aligned rows", f, ql=torch.zeros(2 * 16 * 512 + 1, dtype=BF16)[1:].view(ql.shape))
    refuses("latent must have 16-byte aligned rows", f,
            cache=pca.LatentCache(torch.zeros((4, 16, 514), dtype=BF16)[..., :512], c.rope))
    refuses("out must have 16-byte aligned rows", f, out=odd[..., :512])
    refuses("GPU tensor", f)


def test_decode_entry_refusals():
    L = _lib.lib()

    def call(dtype=_lib.BF16, batch=2, new=1, heads=16, dl=512, dr=64, cache_dtype=_lib.BF16, ql=FAKE, page=16,
             max_pages=40, qlh=512, ws=None, ws_bytes=0, scale=None):
        return L.pcamd_latent_decode(ql, FAKE, dtype, batch, new, heads, dl, dr, 8192, 8192, qlh, 1024, 1024, 64, FAKE,
                                     cache_dtype, 8192, 512, FAKE, 1024, 64, scale, 64, 4, 100, page, FAKE, 40,
                                     max_pages, FAKE, FAKE, 8192, 8192, 512, None, 0, 0, 0, 0.1, ws, ws_bytes, None)

    need = L.pcamd_latent_decode_workspace(2, 1, 16, 512, 16, 40)
    assert need > 0
    for kw, code, text in (({"dtype": _lib.F32}, _lib.ERR_INVALID, b"bf16 or fp16"),
                           ({"cache_dtype": _lib.F16}, _lib.ERR_INVALID, b"cache holds"),
                           ({"dl": 128}, _lib.ERR_UNSUPPORTED, b"512 or 256"),
                           ({"dr": 32}, _lib.ERR_UNSUPPORTED, b"512 and 64"),
                           ({"batch": -1}, _lib.ERR_INVALID, b"negative"),
                           ({"page": 0}, _lib.ERR_INVALID, b"page size"),
                           ({"max_pages": 2 ** 30}, _lib.ERR_UNSUPPORTED, b"too many"),
                           ({"ql": None}, _lib.ERR_INVALID, b"null"),
                           ({"cache_dtype": _lib.E4M3FN}, _lib.ERR_INVALID, b"null"),
                           ({"qlh": 516}, _lib.ERR_INVALID, b"aligned"),
                           ({}, _lib.ERR_INVALID, b"workspace"),
                           ({"ws": FAKE, "ws_bytes": need - 1}, _lib.ERR_INVALID, b"workspace"),
                           ({"ws": ctypes.c_void_p(0x10008), "ws_bytes": need}, _lib.ERR_INVALID, b"workspace")):
        assert call(**kw) == code, kw
        assert text in L.pcamd_last_error(), kw
    assert call(batch=0) == _lib.OK and call(heads=0) == _lib.OK
    assert L.pcamd_latent_decode_workspace(2, 1, 16, 512, 16, 1) == 0  # nothing to split
    assert L.pcamd_latent_decode_workspace(2, 1, 16, 100, 16, 1) == _lib.ERR_UNSUPPORTED
    assert L.pcamd_latent_decode_workspace(0, 1, 16, 512, 16, 1) == 0


# ---------------------------------------------------------------------------
# prefill
# ---------------------------------------------------------------------------
def test_prefill_refusals():
    t = {"q": torch.zeros((5, 2, 192), dtype=BF16), "k_nope": torch.zeros((6, 2, 128), dtype=BF16),
         "k_rope": torch.zeros((6, 64), dtype=BF16), "v": torch.zeros((6, 2, 128), dtype=BF16),
         "cu_q": torch.tensor([0, 5], dtype=torch.int32), "cu_k": torch.tensor([0, 6], dtype=torch.int32)}

    def f(out=None, **kw):
        return pca.latent_prefill(*{**t, **kw}.values(), out=out)

    refuses("T, H, width", f, q=t["q"][0])
    refuses("T, H, width", f, k_rope=t["q"])
    refuses("do not go together", f, k_nope=t["k_nope"][:, :1])
    refuses("do not go together", f, v=t["v"][:5])
    refuses("do not go together", f, k_rope=t["k_rope"][:5])
    refuses("widths must be one of", f, q=t["q"][..., :128])
    refuses("widths must be one of", f, v=t["v"][..., :64])
    refuses("bfloat16 or float16", f, **{n: t[n].float() for n in ("q", "k_nope", "k_rope", "v")})
    refuses("v must be", f, v=t["v"].half())
    refuses("last dimension", f, v=torch.zeros((6, 128, 2), dtype=BF16).transpose(1, 2))
    refuses("cu_q and cu_k", f, cu_q=t["cu_q"].long())
    refuses("cu_q and cu_k", f, cu_k=t["cu_k"][:1])
    refuses("cu_q and cu_k", f, cu_q=t["cu_q"][:0], cu_k=t["cu_k"][:0])
    refuses("out must be", f, out=t["q"])
    refuses("v must have 16-byte aligned rows", f, v=torch.zeros((6, 2, 132), dtype=BF16)[..., :128])
    refuses("k_rope must have 16-byte aligned rows", f, k_rope=torch.zeros((6, 66), dtype=BF16)[..., :64])
    refuses("GPU tensor", f)


def test_prefill_entry_refusals():
    L = _lib.lib()

    def call(q=FAKE, dtype=_lib.BF16, tq=5, tk=6, heads=2, dn=128, dr=64, dv=128, sqh=192, n=1, cu=FAKE):
        return L.pcamd_latent_prefill(q, FAKE, FAKE, FAKE, dtype, tq, tk, heads, dn, dr, dv, 384, sqh, 256, 128, 64,
                                      256, 128, cu, FAKE, n, FAKE, 256, 128, None, 0, 0, 0.1, 1, None)

    for kw, code, text in (({"dtype": _lib.F32}, _lib.ERR_INVALID, b"bf16 or fp16"),
                           ({"dn": 64}, _lib.ERR_UNSUPPORTED, b"widths"), ({"tq": -1}, _lib.ERR_INVALID, b"negative"),
                           ({"tk": 2 ** 31}, _lib.ERR_UNSUPPORTED, b"tokens"),
                           ({"tq": 2 ** 30, "heads": 128}, _lib.ERR_UNSUPPORTED, b"grid"),
                           ({"q": None}, _lib.ERR_INVALID, b"null"), ({"cu": None}, _lib.ERR_INVALID, b"null"),
                           ({"sqh": 196}, _lib.ERR_INVALID, b"aligned"),
                           ({"q": ctypes.c_void_p(0x10008)}, _lib.ERR_INVALID, b"aligned")):
        assert call(**kw) == code, kw
        assert text in L.pcamd_last_error(), kw
    assert call(tq=0) == _lib.OK and call(heads=0) == _lib.OK
