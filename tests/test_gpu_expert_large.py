"""Rows past the cache and grids past 2^20 workgroups: what the routing kernels and the int8 quantizer do at large
sizes only. Rows of more than 128 MB are stored past the cache by kernels of their own."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca
from test_gpu_expert import U, ids_of, rounded

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_rows_past_the_cache(dev, dtype):
    width = 4096 if dtype == FP32 else 8192
    tokens, choices = 2100, 4
    assert tokens * choices * width * dtype.itemsize > 128 << 20
    plan = pca.expert_sort(ids_of(dev, tokens, choices, 6, none=0.2), 6)
    used = plan.starts[-1].item()
    assert 0 < used < tokens * choices
    token = plan.order[:used].long() // choices
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn((tokens, width), generator=g, device=dev).to(dtype)
    torch.full((tokens * choices, width), float("nan"), dtype=dtype, device=dev)  # what the output's memory may hold
    out = pca.expert_dispatch(x, plan)
    assert torch.equal(out[:used], x[token]) and not out[used:].any()
    rows = torch.randn((tokens * choices, width), generator=g, device=dev).to(dtype).requires_grad_()
    w = torch.rand((tokens, choices), generator=g, device=dev).requires_grad_()
    grad = torch.randn((tokens, width), generator=g, device=dev).to(dtype)
    to_rows, to_weights = torch.autograd.grad(pca.expert_combine(rows, plan, w), (rows, w), grad)
    wd = w.detach().flatten()[plan.order[:used].long()].double()
    want = grad[token].double() * wd[:, None]
    assert ((to_rows[:used].double() - want).abs() <= rounded(dtype, want) + U * want.abs()).all()
    assert not to_rows[used:].any()
    parts = rows.detach()[:used].double() * grad[token].double()
    dots, size = torch.zeros((2, tokens * choices), dtype=torch.float64, device=dev)
    dots[plan.order[:used].long()], size[plan.order[:used].long()] = parts.sum(1), parts.abs().sum(1)
    steps = 2 + 8 + 4 + 6 + 4  # a product, a lane's sums in a pass, the passes, a wave's and the waves'
    assert ((to_weights.flatten().double() - dots).abs() <= steps * U * size).all()


def test_more_tokens_than_a_grid_row(dev):
    tokens, choices, width = 2 ** 20 + 77, 2, 8
    plan = pca.expert_sort(ids_of(dev, tokens, choices, 9), 9)
    used = plan.starts[-1].item()
    flat, token = plan.place.flatten().long(), plan.order.long() // choices
    assert torch.equal(plan.order.sort().values, torch.arange(tokens * choices, device=dev, dtype=torch.int32))
    assert torch.equal(torch.where(flat < 0, -1 - flat, flat)[plan.order.long()], torch.arange(tokens * choices, device=dev))
    x = torch.randn((tokens, width), device=dev).to(BF16).requires_grad_()
    out = pca.expert_dispatch(x, plan)
    assert torch.equal(out[:used], x.detach()[token[:used]]) and not out[used:].any()
    w = torch.rand((tokens, choices), device=dev).requires_grad_()
    rows = torch.randn((tokens * choices, width), device=dev).to(BF16).requires_grad_()
    y = pca.expert_combine(rows, plan, w)
    kept = (flat >= 0).view(tokens, choices, 1)
    parts = torch.where(kept, rows.detach().double()[plan.place.clamp(min=0).long()] * w.detach().double()[..., None], 0.0)
    want, size = parts.sum(1), parts.abs().sum(1)
    assert ((y.double() - want).abs() <= rounded(BF16, want) + 4 * U * size).all()
    g = torch.randn((tokens, width), device=dev).to(BF16)
    to_rows, to_weights = torch.autograd.grad(y, (rows, w), g)
    want = g.double()[token[:used]] * w.detach().double().flatten()[plan.order[:used].long()][:, None]
    assert ((to_rows[:used].double() - want).abs() <= rounded(BF16, want) + U * want.abs()).all()
    assert not to_rows[used:].any()
    parts = torch.where(kept, rows.detach().double()[plan.place.clamp(min=0).long()] * g.double()[:, None], 0.0)
    assert ((to_weights.double() - parts.sum(-1)).abs() <= (2 + 8 + 1 + 6 + 4) * U * parts.abs().sum(-1)).all()
    back, = torch.autograd.grad(out, x, to_rows)
    parts = torch.where(kept, to_rows.double()[plan.place.clamp(min=0).long()], 0.0)
    want, size = parts.sum(1), parts.abs().sum(1)
    assert ((back.double() - want).abs() <= rounded(BF16, want) + 3 * U * size).all()


@pytest.mark.parametrize("rows,n", [(2 ** 22 + 9, 16), (2 ** 20 + 3, 2056)])
def test_more_rows_than_a_grid_row(dev, rows, n):
    """A wave a row and a workgroup a row; each result equals that of the call's two halves, which fit."""
    x = torch.randn((rows, n), dtype=BF16, device=dev)
    q = pca.int8_quant(x)
    half = rows // 2
    for part in (slice(0, half), slice(half, rows)):
        p = pca.int8_quant(x[part])
        assert torch.equal(q.tensor[part], p.tensor) and torch.equal(q.dequant_scale[part], p.dequant_scale)
