"""What the int8 products and the experts' operators refuse, on the CPU (no
kernel is launched on these paths)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd import _lib

BF16 = torch.bfloat16
FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first


def refuses(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def codes(shape, axis, *, scale=None, dtype=torch.int8):
    """Codes of the shape with scales of rows (-2) or columns (-1); columns lie K-major."""
    if axis == -1:
        t = torch.zeros((*shape[:-2], shape[-1], shape[-2]), dtype=dtype).transpose(-1, -2)
        s = torch.ones((*shape[:-2], shape[-1]))
    else:
        t, s = torch.zeros(shape, dtype=dtype), torch.ones(shape[:-1])
    return pca.QuantResult(t, s if scale is None else scale, "x", "channel", {"channel_axis": axis})


def plan(tokens=4, choices=2, experts=3, **over):
    parts = {"order": torch.zeros(tokens * choices, dtype=torch.int32),
             "place": torch.zeros((tokens, choices), dtype=torch.int32),
             "starts": torch.zeros(experts + 1, dtype=torch.int32), **over}
    return pca.ExpertPlan(**parts)


def test_quant_refusals():
    x, f = torch.zeros((4, 32), dtype=BF16), pca.int8_quant
    refuses("2D or 3D", f, x[0])
    refuses("channel_axis", f, x, channel_axis=0)
    refuses("input dtype", f, x.double())
    refuses("eps", f, x, eps=-1.0)
    refuses("eps", f, x, eps=float("nan"))
    refuses("contiguous along", f, x.t())
    refuses("contiguous along", f, x, channel_axis=-1)
    refuses("GPU tensor", f, x)
    refuses("GPU tensor", f, x.t(), channel_axis=-1)


def test_bmm_refusals():
    f = pca.int8_bmm
    a, b = codes((2, 4, 32), -2), codes((2, 32, 6), -1)
    refuses("3D", f, codes((4, 32), -2), b)
    refuses("activation", f, a, b, activation="relu")
    refuses("int8 tensors", f, codes((2, 4, 32), -2, dtype=torch.uint8), b)
    refuses("shape mismatch", f, a, codes((2, 16, 6), -1))
    refuses("shape mismatch", f, a, codes((1, 32, 6), -1))
    refuses("contiguous along K", f, a, pca.QuantResult(b.tensor.contiguous(), b.dequant_scale, "x", "channel", b.meta))
    refuses("halves", f, a, codes((2, 32, 7), -1), activation="swiglu")
    refuses("out_dtype", f, a, b, out_dtype=torch.float8_e4m3fn)
    refuses("channel_axis=-2", f, pca.QuantResult(a.tensor, a.dequant_scale, "x", "channel", {"channel_axis": -1}), b)
    refuses("shape", f, codes((2, 4, 32), -2, scale=torch.ones(2, 5)), b)
    refuses("float32", f, codes((2, 4, 32), -2, scale=torch.ones(2, 4).double()), b)
    refuses("out must have shape", f, a, b, out=torch.zeros((2, 4, 5), dtype=BF16))
    refuses("out must have dtype", f, a, b, out=torch.zeros((2, 4, 6)))
    refuses("bias must have shape", f, a, b, bias=torch.zeros(6))
    refuses("bias dtype", f, a, b, bias=torch.zeros((2, 4, 6), dtype=torch.float64))
    refuses("K must be at most 131071", f, codes((1, 1, 131072), -2), codes((1, 131072, 1), -1))
    refuses("GPU tensor", f, a, b)


def test_sort_refusals():
    ids, f = torch.zeros((4, 2), dtype=torch.int32), pca.expert_sort
    refuses("ids must be", f, ids[0], 3)
    refuses("ids must be", f, ids.float(), 3)
    refuses("ids must be", f, ids.t(), 3)
    refuses("experts must be", f, ids, 0)
    refuses("experts must be", f, ids, 1025)
    refuses("choices", f, torch.zeros((1, 129), dtype=torch.int64), 3)
    refuses("GPU tensor", f, ids, 3)


def test_row_refusals():
    x, rows, w, p = torch.zeros((4, 8)), torch.zeros((8, 8)), torch.zeros((4, 2)), plan()
    refuses("x must be", pca.expert_dispatch, x[:3], p)
    refuses("x must be", pca.expert_dispatch, x[0], p)
    refuses("float32, bfloat16", pca.expert_dispatch, x.double(), p)
    refuses("last dimension", pca.expert_dispatch, torch.zeros((8, 4)).t(), p)
    refuses("place must be", pca.expert_dispatch, x, plan(place=torch.zeros((4, 2), dtype=torch.int64)))
    refuses("GPU tensor", pca.expert_dispatch, x, p)
    refuses("rows must be", pca.expert_combine, x, p, w)
    refuses("weights must be", pca.expert_combine, rows, p, w[:3])
    refuses("weights must be", pca.expert_combine, rows, p, w.double())
    refuses("weights must be", pca.expert_combine, rows, p, torch.zeros((2, 4)).t())
    refuses("last dimension", pca.expert_combine, rows.t(), p, w)
    refuses("GPU tensor", pca.expert_combine, rows, p, w)


def test_expert_bmm_refusals():
    f, p = pca.expert_bmm, plan()
    a, b = codes((8, 32), -2), codes((3, 32, 6), -1)
    refuses(r"A must be \[rows, K\]", f, codes((1, 8, 32), -2), b, p)
    refuses("int8 tensors", f, a, codes((3, 32, 6), -1, dtype=torch.uint8), p)
    refuses("shape mismatch", f, a, codes((3, 16, 6), -1), p)
    refuses("plan must be of 2 experts", f, a, codes((2, 32, 6), -1), p)
    refuses("plan must be", f, a, b, plan(order=torch.zeros(7, dtype=torch.int32)))
    refuses("place must be", f, a, b, plan(place=torch.zeros((8, 2), dtype=torch.int32).t()))
    refuses("4 rows with gather=True", f, a, b, p, gather=True)
    refuses("8 rows with gather=False", f, codes((4, 32), -2), b, p)
    refuses("bias must be", f, a, b, p, bias=torch.zeros((3, 5)))
    refuses("out must be", f, a, b, p, out=torch.zeros((8, 5), dtype=BF16))
    refuses("last dimension", f, a, b, p, out=torch.zeros((6, 8), dtype=BF16).t())
    refuses("halves", f, a, codes((3, 32, 7), -1), p, activation="swiglu")
    refuses("GPU tensor", f, a, b, p)


def test_entry_refusals():
    L = _lib.lib()

    def says(rc, want, text):
        assert rc == want and text in L.pcamd_last_error(), (rc, L.pcamd_last_error())

    def quant(dtype=_lib.BF16, m=4, n=40, y=FAKE, sym=48, eps=1e-12, x=FAKE):
        return L.pcamd_quant_int8(x, dtype, 1, m, n, 0, 40, y, 0, sym, FAKE, 0, 1, eps, None)

    says(quant(dtype=3), -1, b"input dtype")
    says(quant(m=-1), -1, b"negative")
    says(quant(eps=float("nan")), -1, b"eps")
    says(quant(y=None), -1, b"null")
    says(quant(sym=40), -1, b"16-byte aligned")
    says(quant(x=ctypes.c_void_p(0x10001)), -1, b"aligned to its elements")
    says(quant(n=2**31), -2, b"more than")
    assert quant(m=0) == 0

    def bmm(m=4, n=8, k=32, sam=32, a=FAKE, c_dtype=_lib.BF16, act=0, batch=1, sab=0):
        return L.pcamd_bmm_int8(a, FAKE, batch, m, n, k, sab, sam, 0, 32, FAKE, c_dtype, 0, 8, None, 0, 0, 0, 0,
                                FAKE, 0, 1, FAKE, 0, 1, act, None)

    says(bmm(m=-1), -1, b"negative")
    says(bmm(c_dtype=3), -1, b"output dtype")
    says(bmm(act=9), -1, b"activation")
    says(bmm(k=131072, sam=131072), -2, b"131071")
    says(bmm(a=ctypes.c_void_p(0x10008)), -1, b"rows of a")
    says(bmm(sam=40), -1, b"rows of a")
    says(bmm(sam=16), -1, b"not overlap")
    says(bmm(batch=2, sab=8), -1, b"multiples of 16")
    says(bmm(a=None), -1, b"null")
    assert bmm(m=0) == 0 and bmm(n=0) == 0 and bmm(batch=0) == 0

    says(L.pcamd_expert_sort_workspace(10, 1025), -2, b"experts")
    says(L.pcamd_expert_sort_workspace(-1, 8), -1, b"negative")
    need = L.pcamd_expert_sort_workspace(100000, 8)
    assert need > 0 and L.pcamd_expert_sort_workspace(4096, 8) == 0
    says(L.pcamd_expert_sort(FAKE, 2, 10, 8, FAKE, FAKE, FAKE, None, 0, None), -1, b"int32 or int64")
    says(L.pcamd_expert_sort(FAKE, 4, 10, 8, None, FAKE, FAKE, None, 0, None), -1, b"null")
    says(L.pcamd_expert_sort(FAKE, 4, 100000, 8, FAKE, FAKE, FAKE, FAKE, need - 1, None), -1, b"workspace")

    says(L.pcamd_expert_dispatch(FAKE, 3, 4, 2, 8, 8, FAKE, FAKE, 8, None), -1, b"rows must be")
    says(L.pcamd_expert_dispatch(FAKE, 0, 4, 129, 8, 8, FAKE, FAKE, 8, None), -2, b"128 choices")
    says(L.pcamd_expert_dispatch(FAKE, 0, 2**30, 2, 8, 8, FAKE, FAKE, 8, None), -2, b"2^31 - 1 pairs")
    says(L.pcamd_expert_combine(FAKE, 0, 4, 2, 8, 8, FAKE, FAKE, 3, FAKE, 8, None), -1, b"weights must be")
    says(L.pcamd_expert_combine(FAKE, 0, 4, 2, 8, 8, FAKE, FAKE, 0, None, 8, None), -1, b"null")
    says(L.pcamd_expert_combine_backward(None, FAKE, 0, 4, 2, 8, 8, 8, FAKE, FAKE, 0, FAKE, 8, None, None), -1, b"null")

    def grouped(a_rows=8, order=None, pairs=8, choices=2, sam=32, starts=FAKE):
        return L.pcamd_expert_bmm_int8(FAKE, a_rows, FAKE, 3, 8, 32, sam, 256, 32, FAKE, _lib.BF16, 8, None, 0, 0, 0,
                                       FAKE, 1, FAKE, 8, 1, starts, order, pairs, choices, 0, None)

    says(grouped(a_rows=4), -1, b"do not go with")
    says(grouped(order=FAKE), -1, b"do not go with")
    says(grouped(a_rows=8, order=FAKE, choices=0), -1, b"do not go with")
    says(grouped(starts=None), -1, b"null")
    says(grouped(sam=24), -1, b"rows of a")
    assert grouped(a_rows=0, pairs=0) == 0


def test_row_entries_refuse_the_widest_rows():
    """A thread steps on past the row's end by up to 64 * 256 columns, which has to fit 32 bits."""
    L = _lib.lib()
    for width, rc in ((2**31 - 65537, -1), (2**31 - 65536, -2), (2**31 - 8192, -2)):  # -1: null pointers, seen later
        assert L.pcamd_expert_dispatch(None, _lib.BF16, 1, 1, width, width, FAKE, None, width, None) == rc
        assert L.pcamd_expert_combine(None, _lib.BF16, 1, 1, width, width, FAKE, FAKE, 0, None, width, None) == rc
