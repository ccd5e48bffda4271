"""Forward-mode derivatives of expert_dispatch and expert_combine on the GPU."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import practice_cuda_amd as pca
from practice_cuda_amd.expert_layer import ExpertMLP

pytestmark = pytest.mark.gpu


def tangent_of(fn, *pairs):
    with forward_ad.dual_level():
        return forward_ad.unpack_dual(fn(*[v if t is None else forward_ad.make_dual(v, t) for v, t in pairs])).tangent


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("needs_grad", [False, True])
def test_tangents(dev, dtype, needs_grad):
    """Both operators are linear in each input, so a tangent is the operator's result with the tangent in its place."""
    g = torch.Generator(device=dev).manual_seed(3)
    plan = pca.expert_sort(torch.randint(-1, 5, (50, 3), generator=g, device=dev), 5)
    x, xt = (torch.randn((50, 72), generator=g, device=dev).to(dtype) for _ in range(2))
    rows, rt = (torch.randn((150, 72), generator=g, device=dev).to(dtype) for _ in range(2))
    w, wt = (torch.randn((50, 3), generator=g, device=dev) for _ in range(2))
    along_rows, along_w = pca.expert_combine(rt, plan, w), pca.expert_combine(rows, plan, wt)
    moved = pca.expert_dispatch(xt, plan)
    for t in (x, rows, w):
        t.requires_grad_(needs_grad)
    assert torch.equal(tangent_of(lambda x: pca.expert_dispatch(x, plan), (x, xt)), moved)

    def f(rows, w):
        return pca.expert_combine(rows, plan, w)

    assert torch.equal(tangent_of(f, (rows, rt), (w, None)), along_rows)
    assert torch.equal(tangent_of(f, (rows, None), (w, wt)), along_w)
    assert torch.equal(tangent_of(f, (rows, rt), (w, wt)), along_rows + along_w)


def test_the_layers(dev):
    """The trained layer's tangents against differences (it is smooth, and fp32 sums of up to 100 products of unit size
    round by about 1e-5; a central difference of step 1e-2 leaves about 1e-4 of a third derivative of unit size); the
    served one has none for its tokens."""
    torch.manual_seed(2)
    layer = ExpertMLP(32, 16, 3, device=dev, dtype=torch.float32)
    x, xt = torch.randn((20, 32), device=dev), torch.randn((20, 32), device=dev)
    ids, w = torch.randint(-1, 3, (20, 2), device=dev), torch.rand((20, 2), device=dev)
    with torch.no_grad():
        got = tangent_of(lambda x: layer(x, ids, w), (x, xt))
        want = (layer(x + 1e-2 * xt, ids, w) - layer(x - 1e-2 * xt, ids, w)) / 2e-2
    assert (got - want).norm() <= 2e-3 * want.norm()
    served = layer.served()
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        tangent_of(lambda x: served(x, ids, w), (x.bfloat16(), xt.bfloat16()))
