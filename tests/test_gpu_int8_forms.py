"""Every form of the int8 products at every kind of size, on the GPU.

The entries choose a form by the sizes' modelled time, so the tiled forms run at large sizes only, where ends of tiles,
groups and inner sizes are few. Here each form is asked for by name and compared with 64 bits under the bounds that
the other tests of these products derive. Accesses past the operands would not show in the values: the outputs lie
between guards, and rows, columns and bytes behind the operands' ends hold codes that would change the sums."""
from __future__ import annotations

import math

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd import _lib
from test_gpu_expert import ids_of
from test_gpu_int8 import check_product

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
FORMS = range(9)
TILED = (7, 8)
UNGATED = (0, 3)  # a column block of 16 has no room for gates and others


@pytest.fixture
def use(monkeypatch):
    """use(form): the products that follow take it."""
    L, launch = _lib.lib(), _lib.launch
    forced = {"pcamd_bmm_int8": L.pcamd_selftest_bmm_int8, "pcamd_expert_bmm_int8": L.pcamd_selftest_expert_bmm_int8}

    def by(form):
        def launch_form(fn, t, *args):
            test = forced.get(fn.__name__)
            return launch(fn, t, *args) if test is None else launch(lambda *a: test(form, *a), t, *args)

        monkeypatch.setattr(_lib, "launch", launch_form)

    return by


def operand(g, shape):
    """Codes of the whole range between other codes: rows and bytes behind their ends. Scales around one."""
    rows, k = shape[-2:]
    wide = torch.randint(-128, 128, (*shape[:-2], rows + 2, -(-k // 16) * 16 + 16), generator=g, device=g.device,
                         dtype=torch.int8)
    return wide[..., 1:rows + 1, :k], torch.rand(shape[:-1], generator=g, device=g.device) + 0.5


def quantized(t, scale, axis):
    return pca.QuantResult(t if axis == -2 else t.transpose(-1, -2), scale, "x", "channel", {"channel_axis": axis})


def guarded(dev, shape, dtype):
    wide = torch.full((*shape[:-2], shape[-2] + 2, shape[-1] + 11), 7.0, dtype=dtype, device=dev)
    return wide, wide[..., 1:-1, 5:shape[-1] + 5]


def product(dev, batch, m, n, k, *, out=FP32, activation="none", bias=None):
    """n: columns of B"""
    g = torch.Generator(device=dev).manual_seed(1000 * m + 10 * n + k)
    (a, sa), (w, sw) = operand(g, (batch, m, k)), operand(g, (batch, n, k))
    sa = sa / (74.0 * 74.0 * math.sqrt(max(k, 1)))  # outputs of about unit size
    if bias is not None:
        bias = torch.randn((batch, m if bias == "rows" else 1, n), generator=g, device=dev).to(BF16).expand(-1, m, -1)
    wide, y = guarded(dev, (batch, m, n // 2 if activation == "swiglu" else n), out)
    pca.int8_bmm(quantized(a, sa, -2), quantized(w, sw, -1), out_dtype=out, bias=bias, activation=activation, out=y)
    acc = torch.matmul(a.double(), w.double().transpose(1, 2).contiguous())
    check_product(y, acc, sa.double().unsqueeze(-1) * sw.double().unsqueeze(1), bias, activation)
    y.fill_(7.0)
    assert (wide == 7.0).all()


@pytest.mark.parametrize("k", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 320, 1031, 2064])
@pytest.mark.parametrize("form", FORMS)
def test_inner(dev, use, form, k):
    use(form)
    for m, n in ((1, 1), (19, 37), (131, 259)):
        product(dev, 1, m, n, k)


@pytest.mark.parametrize("m", [1, 15, 16, 17, 63, 65, 127, 128, 129, 255, 256, 257, 511, 700])
@pytest.mark.parametrize("form", FORMS)
def test_rows_and_columns(dev, use, form, m):
    use(form)
    for n in (1, 3, 16, 127, 129, 255, 257, 530):
        product(dev, 1, m, n, 272, out=FP16)


@pytest.mark.parametrize("out", [BF16, FP16, FP32])
@pytest.mark.parametrize("activation", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("bias", [None, "one", "rows"])
@pytest.mark.parametrize("form", FORMS)
def test_epilogue(dev, use, form, bias, activation, out):
    use(form)
    if form in UNGATED and activation == "swiglu":
        with pytest.raises(ValueError, match="does not take"):
            product(dev, 1, 4, 4, 16, activation=activation)
        return
    for m, n, k in ((3, 2, 40), (270, 514, 400), (150, 254, 128)):
        product(dev, 2, m, n, k, out=out, activation=activation, bias=bias)


@pytest.mark.parametrize("form", FORMS)
def test_batches(dev, use, form):
    use(form)
    product(dev, 5, 130, 200, 257)
    product(dev, 70, 17, 33, 64)
    product(dev, 2, 600, 700, 512, out=BF16)


@pytest.mark.parametrize("form", TILED)
def test_many_tiles(dev, use, form):
    """More row tiles than a group of eight, with a rest; more tiles than CUs."""
    use(form)
    product(dev, 1, 2600, 1300, 96, out=BF16)
    product(dev, 1, 130, 9000, 200, out=BF16)
    product(dev, 1, 4700, 5200, 64, out=BF16)
    product(dev, 1, 2100, 2060, 160, out=BF16, activation="swiglu")


@pytest.mark.parametrize("form", TILED)
def test_no_inner_size_is_refused(dev, use, form):
    use(form)
    with pytest.raises(ValueError, match="does not take"):
        product(dev, 1, 4, 4, 0)


def test_longest_sums(dev, use):
    """The largest sum, in every form: each product 128 * 128, k = 131071."""
    a = torch.full((1, 3, 131072), -128, dtype=torch.int8, device=dev)[..., :131071]
    one = torch.ones((1, 3), device=dev)
    for form in FORMS:
        use(form)
        y = pca.int8_bmm(quantized(a, one, -2), quantized(a, one, -1), out_dtype=FP32)
        assert (y == float(128 * 128 * 131071)).all(), form


# ---------------------------------------------------------------------------
# grouped
# ---------------------------------------------------------------------------
def grouped(dev, ids, experts, n, k, *, gather, out=FP32, activation="none", bias=False):
    g = torch.Generator(device=dev).manual_seed(ids.numel() + 10 * n + k)
    plan = pca.expert_sort(ids, experts)
    pairs, choices = ids.numel(), ids.shape[1]
    (a, sa), (w, sw) = operand(g, (ids.shape[0] if gather else pairs, k)), operand(g, (experts, n, k))
    sa = sa / (74.0 * 74.0 * math.sqrt(k))
    bias = torch.randn((experts, n), generator=g, device=dev).to(FP16) if bias else None
    wide, y = guarded(dev, (pairs, n // 2 if activation == "swiglu" else n), out)
    pca.expert_bmm(quantized(a, sa, -2), quantized(w, sw, -1), plan, gather=gather, out_dtype=out, bias=bias,
                   activation=activation, out=y)
    starts = plan.starts.tolist()
    assert not y[starts[-1]:].any()
    rows = plan.order.long() // choices if gather else torch.arange(pairs, device=dev)
    for e in range(experts):
        lo, hi = starts[e], starts[e + 1]
        if hi > lo:
            at = rows[lo:hi]
            acc = torch.matmul(a[at].double(), w[e].double().t().contiguous())
            check_product(y[lo:hi], acc, sa[at].double()[:, None] * sw[e].double(),
                          None if bias is None else bias[e].expand(hi - lo, -1), activation)
    y.fill_(7.0)
    assert (wide == 7.0).all()


SIZES = [0, 1, 15, 16, 17, 0, 63, 64, 65, 127, 128, 129, 0, 255, 256, 257, 2, 383, 385, 513, 0]  # rows of the experts


def of_sizes(dev, sizes, none=0, seed=1):
    """ids [T, 1] that give the experts these sizes, shuffled, and `none` tokens without one"""
    ids = torch.repeat_interleave(torch.arange(-1, len(sizes), device=dev), torch.tensor([none, *sizes], device=dev))
    g = torch.Generator(device=dev).manual_seed(seed)
    return ids[torch.randperm(ids.numel(), generator=g, device=dev)].int()[:, None].contiguous()


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("none", [0, 1, 300])
@pytest.mark.parametrize("form", FORMS)
def test_group_ends(dev, use, form, none, gather):
    use(form)
    grouped(dev, of_sizes(dev, SIZES, none), len(SIZES), 150, 208, gather=gather)


@pytest.mark.parametrize("k", [1, 16, 17, 63, 65, 127, 129, 191, 193, 257, 1031])
@pytest.mark.parametrize("form", FORMS)
def test_group_inner(dev, use, form, k):
    use(form)
    grouped(dev, ids_of(dev, 150, 3, 4), 4, 70, k, gather=True)
    grouped(dev, ids_of(dev, 400, 2, 3), 3, 270, k, gather=False)


@pytest.mark.parametrize("out", [BF16, FP16, FP32])
@pytest.mark.parametrize("activation", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_group_epilogue(dev, use, form, bias, activation, out):
    if form in UNGATED and activation == "swiglu":
        return
    use(form)
    for n in (2, 258, 514):
        grouped(dev, ids_of(dev, 500, 2, 4), 4, n, 200, gather=True, out=out, activation=activation, bias=bias)


@pytest.mark.parametrize("form", FORMS)
def test_few_of_many(dev, use, form):
    """More experts than a wave's lanes, most without rows; all rows at one expert, at the last, at none."""
    use(form)
    grouped(dev, ids_of(dev, 40, 2, 200), 200, 33, 80, gather=True)
    grouped(dev, ids_of(dev, 1000, 4, 130), 130, 48, 64, gather=True)
    for value in (0, 69, -1):
        ids = torch.full((300, 2), value, dtype=torch.int32, device=dev)
        grouped(dev, ids, 70, 40, 96, gather=True)
        grouped(dev, ids, 70, 40, 96, gather=False)


@pytest.mark.parametrize("form", TILED)
def test_many_group_tiles(dev, use, form):
    use(form)
    grouped(dev, ids_of(dev, 3000, 3, 20), 20, 600, 96, gather=True, out=BF16)
    grouped(dev, ids_of(dev, 2000, 8, 128), 128, 300, 128, gather=True, out=BF16, activation="swiglu")
    # most pairs are another rank's experts
    grouped(dev, ids_of(dev, 4000, 4, 16, none=0.9), 16, 300, 128, gather=True, out=BF16)
