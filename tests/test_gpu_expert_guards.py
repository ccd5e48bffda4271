"""Plans that are none leave everything but their outputs alone, and gradients of strided rows whole, row by row."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd import _lib
from test_gpu_expert import codes, ids_of

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def bad_plans(good):
    order, place, starts = good.order, good.place, good.starts
    yield pca.ExpertPlan(order + 1000, place + 70, starts * 3)
    yield pca.ExpertPlan(order - 1000, -1 - place - 70, starts - 50)
    yield pca.ExpertPlan(torch.full_like(order, 2**31 - 1), torch.full_like(place, 2**31 - 1), starts.flip(0).contiguous())
    yield pca.ExpertPlan(torch.full_like(order, -2**31), torch.full_like(place, -2**31), torch.full_like(starts, 2**31 - 1))
    yield pca.ExpertPlan(order.zero_().clone(), torch.zeros_like(place), torch.full_like(starts, -2**31))


def guarded(rows, width, dtype, dev):
    wide = torch.full((rows + 2, width), 7.0, dtype=dtype, device=dev)
    return wide, wide[1:-1]


def kept(wide):
    return bool((wide[0] == 7.0).all() and (wide[-1] == 7.0).all())


@pytest.mark.parametrize("width", [64, 13])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rows(dev, dtype, width):
    L, code = _lib.lib(), _lib.dtype_code(dtype)
    tokens, choices = 40, 2
    pairs = tokens * choices
    x, rows = torch.ones((tokens, width), dtype=dtype, device=dev), torch.ones((pairs, width), dtype=dtype, device=dev)
    w = torch.ones((tokens, choices), device=dev)
    for plan in bad_plans(pca.expert_sort(ids_of(dev, tokens, choices, 4, none=0.0), 4)):
        place = plan.place.data_ptr()
        wide, out = guarded(pairs, width, dtype, dev)
        rc = _lib.launch(L.pcamd_expert_dispatch, x, x.data_ptr(), code, tokens, choices, width, width, place,
                         out.data_ptr(), width)
        assert rc == 0 and kept(wide)
        wide, out = guarded(tokens, width, dtype, dev)
        rc = _lib.launch(L.pcamd_expert_combine, x, rows.data_ptr(), code, tokens, choices, width, width, place,
                         w.data_ptr(), _lib.F32, out.data_ptr(), width)
        assert rc == 0 and kept(wide)
        wide, out = guarded(pairs, width, dtype, dev)
        wide_w, to_w = guarded(tokens, choices, FP32, dev)
        rc = _lib.launch(L.pcamd_expert_combine_backward, x, x.data_ptr(), rows.data_ptr(), code, tokens, choices, width,
                         width, width, place, w.data_ptr(), _lib.F32, out.data_ptr(), width, to_w.data_ptr())
        assert rc == 0 and kept(wide) and kept(wide_w)


@pytest.mark.parametrize("form", range(9))
@pytest.mark.parametrize("gather", [False, True])
def test_products(dev, monkeypatch, form, gather):
    L, launch = _lib.lib(), _lib.launch
    monkeypatch.setattr(_lib, "launch", lambda fn, t, *args: launch(
        lambda *a: L.pcamd_selftest_expert_bmm_int8(form, *a) if fn.__name__ == "pcamd_expert_bmm_int8" else fn(*a),
        t, *args))
    g = torch.Generator(device=dev).manual_seed(1)
    tokens, choices = 300, 2
    a, sa = codes(g, (tokens if gather else tokens * choices, 64))
    w, sw = codes(g, (4, 32, 64))
    for plan in bad_plans(pca.expert_sort(ids_of(dev, tokens, choices, 4, none=0.0), 4)):
        wide, out = guarded(tokens * choices, 32, BF16, dev)
        pca.expert_bmm(pca.QuantResult(a, sa, "x", "channel", {"channel_axis": -2}),
                       pca.QuantResult(w.transpose(1, 2), sw, "x", "channel", {"channel_axis": -1}), plan,
                       gather=gather, out=out)
        assert kept(wide)


def test_gradient_of_strided_rows(dev):
    """Every row of the gradient: each element is one product, rounded once."""
    plan = pca.expert_sort(ids_of(dev, 30, 2, 4), 4)
    rows = torch.randn((60, 320), device=dev).to(BF16)[:, 3:303].requires_grad_()
    w = torch.rand((30, 2), device=dev)
    g = torch.randn((300, 30), device=dev).to(BF16).t()  # not contiguous along its rows
    back, = torch.autograd.grad(pca.expert_combine(rows, plan, w), rows, g)
    want = torch.zeros((60, 300), dtype=BF16, device=dev)
    used = plan.place.flatten() >= 0
    want[plan.place.flatten()[used].long()] = (g.float().unsqueeze(1) * w.unsqueeze(-1)).flatten(0, 1)[used].to(BF16)
    assert used.any() and not used.all() and torch.equal(back, want)
