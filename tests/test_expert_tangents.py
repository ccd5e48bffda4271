"""Forward-mode derivatives of expert_dispatch and expert_combine, on the CPU: plain torch stands in for the kernels'
launches, so what runs here is how tangents and gradients travel through the operators."""
from __future__ import annotations

import gc
import weakref

import pytest
import torch
from torch.autograd import forward_ad

import practice_cuda_amd as pca
from practice_cuda_amd.impls import hip_expert


@pytest.fixture
def plan(monkeypatch):
    def dispatch(x, place):
        out = torch.zeros((place.numel(), x.shape[1]), dtype=x.dtype)
        for t in range(place.shape[0]):
            for s in place[t].tolist():
                if s >= 0:
                    out[s] = x[t]
        return out

    def combine(rows, place, weights):
        out = torch.zeros((place.shape[0], rows.shape[1]), dtype=rows.dtype)
        for t in range(place.shape[0]):
            for j, s in enumerate(place[t].tolist()):
                if s >= 0:
                    out[t] += rows[s] * (1.0 if weights is None else weights[t, j])
        return out

    def plain(fn):  # as a kernel: values alone
        return lambda *args: fn(*[None if a is None else a.detach().clone() for a in args])

    monkeypatch.setattr(hip_expert, "_dispatch", plain(dispatch))
    monkeypatch.setattr(hip_expert, "_combine", plain(combine))
    monkeypatch.setattr(hip_expert._lib, "require_gpu_tensor", lambda t, name: None)
    place = torch.tensor([[2, 0], [-5, 1], [3, -6]], dtype=torch.int32)  # two pairs without an expert
    order = torch.tensor([1, 3, 0, 4, 2, 5], dtype=torch.int32)
    return pca.ExpertPlan(order, place, torch.tensor([0, 2, 4], dtype=torch.int32))


def tangent_of(fn, *pairs):
    with forward_ad.dual_level():
        return forward_ad.unpack_dual(fn(*[v if t is None else forward_ad.make_dual(v, t) for v, t in pairs])).tangent


@pytest.mark.parametrize("needs_grad", [False, True])
def test_dispatch(plan, needs_grad):
    x, xt = torch.randn(3, 4), torch.randn(3, 4)
    got = tangent_of(lambda x: pca.expert_dispatch(x, plan), (x.requires_grad_(needs_grad), xt))
    assert got is not None and torch.equal(got, pca.expert_dispatch(xt, plan))
    with torch.no_grad():
        got = tangent_of(lambda x: pca.expert_dispatch(x, plan), (x, xt))
    assert got is not None and torch.equal(got, pca.expert_dispatch(xt, plan))


@pytest.mark.parametrize("needs_grad", [False, True])
def test_combine(plan, needs_grad):
    rows, rows_t, w, w_t = torch.randn(6, 4), torch.randn(6, 4), torch.rand(3, 2), torch.randn(3, 2)
    of_rows, of_weights = pca.expert_combine(rows_t, plan, w), pca.expert_combine(rows, plan, w_t)
    rows.requires_grad_(needs_grad)

    def f(rows, w):
        return pca.expert_combine(rows, plan, w)

    for pair_r, pair_w, want in (((rows, rows_t), (w, None), of_rows), ((rows, None), (w, w_t), of_weights),
                                 ((rows, rows_t), (w, w_t), of_rows + of_weights)):
        got = tangent_of(f, pair_r, pair_w)
        assert got is not None and torch.equal(got, want)


def test_tangents_that_are_not_plain(plan):
    """Transposed, lazily negated and lazily zero tangents."""
    x, wide = torch.randn(3, 4), torch.randn(4, 3)
    got = tangent_of(lambda x: pca.expert_dispatch(x, plan), (x, wide.t()))
    assert torch.equal(got, pca.expert_dispatch(wide.t().contiguous(), plan))
    got = tangent_of(lambda x: pca.expert_dispatch(x, plan), (x, torch._neg_view(wide.t().contiguous())))
    assert torch.equal(got, pca.expert_dispatch(-wide.t().contiguous(), plan))
    got = tangent_of(lambda x: pca.expert_dispatch(x, plan), (x, torch._efficientzerotensor((3, 4))))
    assert torch.equal(got, torch.zeros(6, 4))
    w = torch.rand(3, 2)
    got = tangent_of(lambda w: pca.expert_combine(torch.ones(6, 4), plan, w), (w, torch.ones(2, 3).t()))
    assert torch.equal(got, pca.expert_combine(torch.ones(6, 4), plan, torch.ones(3, 2)))


def test_backward_through_a_tangent(plan):
    """combine is bilinear: the tangent along the weights is linear in the rows, and its gradient is theirs."""
    rows, w, w_t = torch.randn(6, 4), torch.rand(3, 2), torch.randn(3, 2)
    x, x_t = torch.randn(3, 4, requires_grad=True), torch.randn(3, 4, requires_grad=True)
    with forward_ad.dual_level():
        out = pca.expert_dispatch(forward_ad.make_dual(x, x_t), plan)
        tangent = forward_ad.unpack_dual(out).tangent
        back, = torch.autograd.grad(tangent.sum(), x_t)
    assert torch.equal(back, pca.expert_combine(torch.ones(6, 4), plan, torch.ones(3, 2)))


def test_the_gradients_have_no_tangent(plan):
    x = torch.randn(3, 4, requires_grad=True)
    with forward_ad.dual_level():
        out = pca.expert_dispatch(forward_ad.make_dual(x, torch.ones(3, 4)), plan)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            out.square().sum().backward()
        rows, w = torch.randn(6, 4), torch.rand(3, 2, requires_grad=True)
        out = pca.expert_combine(forward_ad.make_dual(rows, torch.ones(6, 4)), plan, w)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            out.sum().backward()


def test_nothing_is_kept_beside_the_saved_tensors(plan):
    """What a saved-tensor hook replaces is freed with the caller's last reference, the output still there."""
    x = torch.randn(6, 4, requires_grad=True)
    rows, w = x * 2.0, torch.rand(3, 2)
    last = weakref.ref(rows)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.numpy(force=True).copy(), torch.from_numpy):
        y = pca.expert_combine(rows, plan, w)
    del rows
    gc.collect()
    assert last() is None and y.requires_grad
