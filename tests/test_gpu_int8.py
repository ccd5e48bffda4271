"""int8_quant and int8_bmm on the GPU against their formulas in 64 bits.

Codes have to be equal: the formula's quotient is taken in fp64, where 127 x is
exact and a quotient that is no tie is further from one than fp64 rounds by.
Products: the sum is exact; converting it, the two scales' product and its
multiplication round three times (2^-24 each), a bias once more, the activation
as derived in `tolerance`, and the output by half a step of its type."""
from __future__ import annotations

import math

import pytest
import torch

import practice_cuda_amd as pca

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def formula(x, eps=1e-12):
    """(codes, scales) of the rows of x, in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1).clamp(min=torch.tensor(eps).item())
    top = top.float().double()  # eps is an fp32 number
    codes = torch.round(127.0 * x / top.unsqueeze(-1))
    return codes.to(torch.int8), top / 127.0


def check_quant(x, axis=-2, eps=1e-12):
    q = pca.int8_quant(x, channel_axis=axis, eps=eps)
    rows = x if axis == -2 else x.transpose(-1, -2)
    codes, scale = formula(rows, eps)
    got = q.tensor if axis == -2 else q.tensor.transpose(-1, -2)
    assert got.shape == rows.shape and got.stride(-1) == 1 and got.data_ptr() % 16 == 0
    assert got.shape[-2] == 1 or got.stride(-2) % 16 == 0
    assert torch.equal(got, codes)
    assert (q.dequant_scale.double() - scale).abs().max() <= scale.abs().max() * U
    assert q.granularity == "channel" and q.meta["channel_axis"] == axis
    return q


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("n", [1, 7, 16, 100, 512, 513, 1031, 2048, 2049, 7168, 16384, 20000, 32768, 33000])
def test_quant_lengths(dev, n, dtype):
    g = torch.Generator(device=dev).manual_seed(n)
    check_quant((torch.randn((5, n), generator=g, device=dev) * 3).to(dtype))


@pytest.mark.parametrize("rows", [1, 3, 255, 4097])
def test_quant_rows(dev, rows):
    g = torch.Generator(device=dev).manual_seed(rows)
    check_quant(torch.randn((2, rows, 392), generator=g, device=dev).to(BF16))


def test_quant_views(dev):
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn((3, 40, 1000), generator=g, device=dev).to(BF16)
    check_quant(x[:, :, 3:900])                                    # rows at odd addresses
    check_quant(x[:, ::2, 1:])
    check_quant(x.transpose(0, 1)[:, 1:])
    check_quant(x[:, :1, :5].expand(3, 7, 5))                      # every row the same memory
    check_quant(x.transpose(-1, -2), axis=-1)                      # a weight's columns
    check_quant(x[0, :, 5:].t(), axis=-1)
    assert pca.int8_quant(x[:, :0]).tensor.shape == (3, 0, 1000)
    empty = pca.int8_quant(x[:, :, :0])
    assert empty.tensor.shape == (3, 40, 0) and torch.equal(empty.dequant_scale, torch.full((3, 40), 1e-12, device=dev) / 127)


def test_quant_borders(dev):
    """Values on and next to the borders of two codes: 254 x = (2 q + 1) top exactly, and its neighbours."""
    for dtype in (BF16, FP16, FP32):
        rows = []
        for top in (127.0, 1.0, 254.0, 3.0, 63.5, 1.9921875):
            edge = (torch.arange(-127, 127, device=dev, dtype=torch.float64) + 0.5) * top / 127.0
            x = edge.to(dtype)
            around = [x, torch.nextafter(x.float(), x.float() + 1).to(dtype), torch.nextafter(x.float(), x.float() - 1).to(dtype)]
            row = torch.cat([*around, torch.tensor([top], device=dev, dtype=dtype)]).clamp(-top, top)
            rows.append(row)
        check_quant(torch.stack(rows))
    check_quant(torch.arange(-127, 128, device=dev).float()[None] / 2 + torch.zeros((3, 1), device=dev))


def test_quant_small_and_zero(dev):
    x = torch.randn((6, 300), device=dev)
    x[1] = 0.0
    x[2] *= 1e-15
    x[3] *= 1e-36
    x[4] *= 1e30
    check_quant(x)
    check_quant(x, eps=0.5)
    check_quant(x.to(BF16), eps=1e-37)
    q = pca.int8_quant(x, eps=0.0)
    keep = [0, 2, 3, 4, 5]
    assert torch.equal(q.tensor[keep], formula(x[keep], 0.0)[0])
    assert not q.tensor[1].any() and q.dequant_scale[1] == 0


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("n", [30, 5000, 40000])
def test_quant_not_finite(dev, n, dtype):
    x = torch.randn((4, n), device=dev).to(dtype)
    x[0, n - 1], x[2, 0], x[2, 1] = math.nan, math.inf, -math.inf
    q = pca.int8_quant(x)
    assert torch.equal(q.dequant_scale.isnan(), torch.tensor([True, False, True, False], device=dev))
    assert not q.tensor[[0, 2]].any()
    codes, scale = formula(x[[1, 3]])
    assert torch.equal(q.tensor[[1, 3]], codes)
    w = pca.int8_quant(torch.randn((1, n, 5), device=dev).transpose(-1, -2).contiguous().transpose(-1, -2), channel_axis=-1)
    y = pca.int8_bmm(pca.QuantResult(q.tensor[None], q.dequant_scale[None], "x", "channel", q.meta), w)
    assert y[0, [0, 2]].isnan().all() and not y[0, [1, 3]].isnan().any()


def test_quant_gradient_is_refused(dev):
    x = torch.randn((4, 64), device=dev, requires_grad=True)
    q = pca.int8_quant(x)
    assert torch.equal(q.tensor, formula(x.detach())[0])
    with pytest.raises(RuntimeError, match="no gradient"):
        q.dequant_scale.sum().backward()


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def operand(g, shape, pad=0):
    """Codes of the whole range with rows at multiples of 16 bytes, and scales around one."""
    wide = -(-shape[-1] // 16) * 16 + pad
    t = torch.randint(-128, 128, (*shape[:-1], wide), generator=g, device=g.device, dtype=torch.int8)[..., :shape[-1]]
    return t, torch.rand(shape[:-1], generator=g, device=g.device) + 0.5


def activated(y, activation, d):
    """(activated y, the error that an error d of y becomes, with the function's own: erff and expf are within 4
    units in the last place, and each further operation within half a one)."""
    if activation == "gelu":
        v = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
        return v, 1.13 * d + 8 * U * y.abs()
    if activation == "swiglu":
        n = y.shape[-1] // 2
        gate, up, dg, du = y[..., :n], y[..., n:], d[..., :n], d[..., n:]
        s = gate * torch.sigmoid(gate)
        ds = 1.1 * dg + 16 * U * s.abs()
        return s * up, ds * up.abs() + s.abs() * du + ds * du + 2 * U * (s * up).abs()
    return y, d


def check_product(got, acc, scale, bias, activation):
    """got against the exact sums acc, their scale and the bias (64 bits)."""
    y = acc * scale
    d = 3.01 * U * y.abs()
    if bias is not None:
        y = y + bias.double()
        d = d + 1.01 * U * (y.abs() + d)
    want, d = activated(y, activation, d)
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal
    assert ((got.double() - want).abs() <= 1.01 * d + half * (want.abs() + d).clamp(min=tiny)).all()


def run(dev, batch, m, n, k, *, out=BF16, bias=None, activation="none", pad=0, seed=0):
    g = torch.Generator(device=dev).manual_seed(1000 * m + 10 * n + k + seed)
    a, sa = operand(g, (batch, m, k), pad)
    w, sw = operand(g, (batch, n, k), pad)
    sa = sa / (74.0 * 74.0 * math.sqrt(max(k, 1)))  # outputs of about unit size, where activations bend
    if bias is not None:
        bias = torch.randn((batch, m if bias == "rows" else 1, n), generator=g, device=dev).to(BF16).expand(-1, m, -1)
    y = pca.int8_bmm(pca.QuantResult(a, sa, "x", "channel", {"channel_axis": -2}),
                     pca.QuantResult(w.transpose(1, 2), sw, "x", "channel", {"channel_axis": -1}),
                     out_dtype=out, bias=bias, activation=activation)
    acc = torch.matmul(a.double(), w.double().transpose(1, 2).contiguous())
    scale = sa.double().unsqueeze(-1) * sw.double().unsqueeze(1)
    assert y.dtype == out
    check_product(y, acc, scale, bias, activation)
    return y


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 127, 129, 200, 257, 500])
@pytest.mark.parametrize("n,k", [(300, 512), (1000, 640), (31, 1031)])
def test_bmm_rows(dev, m, n, k):
    run(dev, 1, m, n, k)


@pytest.mark.parametrize("k", [1, 3, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 400, 2047, 5000])
@pytest.mark.parametrize("m", [3, 40, 300])
def test_bmm_inner(dev, m, k):
    run(dev, 1, m, 96, k, out=FP32)


@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 16, 17, 33, 64, 100, 127, 128, 130, 255, 256, 258, 513])
@pytest.mark.parametrize("m", [5, 70, 260])
def test_bmm_columns(dev, m, n):
    run(dev, 1, m, n, 272, out=FP16)


@pytest.mark.parametrize("out", [BF16, FP16, FP32])
@pytest.mark.parametrize("activation", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("bias", [None, "one", "rows"])
@pytest.mark.parametrize("m,n,k", [(7, 70, 200), (50, 258, 300), (300, 514, 384)])
def test_bmm_epilogue(dev, m, n, k, bias, activation, out):
    run(dev, 2, m, n, k, out=out, bias=bias, activation=activation)


@pytest.mark.parametrize("batch,m,n,k", [(3, 9, 40, 100), (5, 130, 200, 257), (70, 17, 33, 64), (2, 600, 700, 512)])
def test_bmm_batches(dev, batch, m, n, k):
    run(dev, batch, m, n, k, pad=16)


@pytest.mark.parametrize("m,n,k", [(1024, 2048, 1024), (2050, 1030, 1040), (515, 4100, 2304), (4096, 512, 8192)])
def test_bmm_large(dev, m, n, k):
    run(dev, 1, m, n, k)
    run(dev, 1, m, n, k, activation="swiglu")


def test_bmm_longest_sums(dev):
    """The largest sum: every product 128 * 128, k = 131071."""
    for m in (2, 130):
        a = torch.full((1, m, 131072), -128, dtype=torch.int8, device=dev)[..., :131071]
        w = torch.full((1, 130, 131072), -128, dtype=torch.int8, device=dev)[..., :131071]
        one = torch.ones((1, 130), device=dev)
        y = pca.int8_bmm(pca.QuantResult(a, torch.ones((1, m), device=dev), "x", "channel", {"channel_axis": -2}),
                         pca.QuantResult(w.transpose(1, 2), one, "x", "channel", {"channel_axis": -1}), out_dtype=FP32)
        assert (y == float(128 * 128 * 131071)).all()  # 2^14 (2^17 - 1): an fp32 number


def test_bmm_layouts(dev):
    g = torch.Generator(device=dev).manual_seed(5)
    a, sa = operand(g, (2, 50, 160))
    w, sw = operand(g, (2, 72, 160))
    qa = pca.QuantResult(a, sa, "x", "channel", {"channel_axis": -2})
    qb = pca.QuantResult(w.transpose(1, 2), sw, "x", "channel", {"channel_axis": -1})
    want = pca.int8_bmm(qa, qb)
    # an output between guards, with odd strides
    wide = torch.full((2, 52, 81), 7.0, dtype=BF16, device=dev)
    got = pca.int8_bmm(qa, qb, out=wide[:, 1:51, 3:75])
    assert torch.equal(got, want) and got.data_ptr() == wide[:, 1:51, 3:75].data_ptr()
    wide[:, 1:51, 3:75] = 7.0
    assert (wide == 7.0).all()
    # operands that are slices, broadcast batches, scales with strides
    big = torch.zeros((2, 60, 320), dtype=torch.int8, device=dev)
    big[:, 5:55, 32:192] = a
    scales = torch.zeros((2, 100), device=dev)
    scales[:, ::2] = sa
    got = pca.int8_bmm(pca.QuantResult(big[:, 5:55, 32:192], scales[:, ::2], "x", "channel", {"channel_axis": -2}), qb)
    assert torch.equal(got, want)
    one = pca.QuantResult(w[:1].expand(2, -1, -1).transpose(1, 2), sw[:1].expand(2, -1), "x", "channel", {"channel_axis": -1})
    assert torch.equal(pca.int8_bmm(qa, one)[0], want[0])
    # rows that are not aligned are refused, and so are rows that overlap
    odd = torch.zeros((2, 50, 176), dtype=torch.int8, device=dev)[..., 8:168]
    with pytest.raises(ValueError, match="16-byte aligned"):
        pca.int8_bmm(pca.QuantResult(odd, sa, "x", "channel", {"channel_axis": -2}), qb)
    with pytest.raises(ValueError, match="not overlap"):
        pca.int8_bmm(pca.QuantResult(a[:, :1].expand(2, 50, 160), sa, "x", "channel", {"channel_axis": -2}), qb)
    # a bias of any strides
    bias = torch.randn((72, 50, 2), generator=g, device=dev).permute(2, 1, 0)
    acc = torch.matmul(a.double(), w.double().transpose(1, 2).contiguous())
    got = pca.int8_bmm(qa, qb, bias=bias, out_dtype=FP32)
    check_product(got, acc, sa.double().unsqueeze(-1) * sw.double().unsqueeze(1), bias, "none")


def test_bmm_empty(dev):
    def shaped(batch, m, n, k):
        a = pca.QuantResult(torch.zeros((batch, m, k), dtype=torch.int8, device=dev), torch.ones((batch, m), device=dev),
                            "x", "channel", {"channel_axis": -2})
        b = pca.QuantResult(torch.zeros((batch, n, k), dtype=torch.int8, device=dev).transpose(1, 2),
                            torch.ones((batch, n), device=dev), "x", "channel", {"channel_axis": -1})
        return pca.int8_bmm(a, b)

    assert shaped(0, 4, 5, 16).shape == (0, 4, 5)
    assert shaped(2, 0, 5, 16).shape == (2, 0, 5)
    assert shaped(2, 4, 0, 16).shape == (2, 4, 0)
    assert torch.equal(shaped(1, 4, 5, 0), torch.zeros((1, 4, 5), dtype=BF16, device=dev))


def test_bmm_padding_does_not_count(dev):
    """What lies behind a row's k bytes may hold anything."""
    g = torch.Generator(device=dev).manual_seed(9)
    for m in (3, 200):
        a, sa = operand(g, (1, m, 133))
        w, sw = operand(g, (1, 150, 133))
        b = pca.QuantResult(w.transpose(1, 2), sw, "x", "channel", {"channel_axis": -1})
        qa = pca.QuantResult(a, sa, "x", "channel", {"channel_axis": -2})
        want = pca.int8_bmm(qa, b)
        torch.as_strided(a, (1, m, 11), (a.stride(0), 144, 1), a.storage_offset() + 133).fill_(99)
        torch.as_strided(w, (1, 150, 11), (w.stride(0), 144, 1), w.storage_offset() + 133).fill_(-77)
        assert torch.equal(pca.int8_bmm(qa, b), want)


def test_graph_and_streams(dev):
    """Captured once and replayed on new inputs; the same call on a side stream."""
    g = torch.Generator(device=dev).manual_seed(11)
    x = torch.randn((1, 33, 700), generator=g, device=dev).to(BF16)
    w = pca.int8_quant(torch.randn((1, 500, 700), generator=g, device=dev).to(BF16).transpose(1, 2), channel_axis=-1)

    def call():
        return pca.int8_bmm(pca.int8_quant(x), w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, call())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device=dev))
        want = call()
        y.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
