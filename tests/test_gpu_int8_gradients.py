"""The int8 products have no gradient: going backward from them is an error, also where what requires one is a scale."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca

pytestmark = pytest.mark.gpu


def parts(dev, *, a_grad=False, b_grad=False):
    x = torch.randn((6, 32), device=dev, requires_grad=a_grad)
    w = torch.randn((3, 24, 32), device=dev, requires_grad=b_grad)
    return pca.int8_quant(x), pca.int8_quant(w.transpose(1, 2), channel_axis=-1)


@pytest.mark.parametrize("a_grad,b_grad", [(True, False), (False, True)])
def test_products_of_codes_that_require_a_gradient(dev, a_grad, b_grad):
    a, b = parts(dev, a_grad=a_grad, b_grad=b_grad)
    one = pca.QuantResult(a.tensor[None], a.dequant_scale[None], "x", "channel", a.meta)
    two = pca.QuantResult(b.tensor[:1], b.dequant_scale[:1], "x", "channel", b.meta)
    plan = pca.expert_sort(torch.randint(0, 3, (6, 1), device=dev), 3)
    for call, out in ((lambda **kw: pca.int8_bmm(one, two, **kw), (1, 6, 24)),
                      (lambda **kw: pca.expert_bmm(a, b, plan, **kw), (6, 24))):
        y = call()
        assert y.requires_grad
        with pytest.raises(RuntimeError, match="no gradient"):
            y.float().sum().backward()
        with pytest.raises(ValueError, match="requires a gradient"):
            call(out=torch.empty(out, dtype=torch.bfloat16, device=dev))
        with torch.no_grad():
            want = call()
            assert torch.equal(want, y) and not want.requires_grad
