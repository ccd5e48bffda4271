"""Tokens without choices, and no tokens, through the experts' product and the layers."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd.expert_layer import ExpertMLP

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,choices", [(3, 0), (0, 2), (0, 0), (70, 0)])
@pytest.mark.parametrize("gather", [True, False])
def test_expert_bmm(dev, tokens, choices, gather):
    plan = pca.expert_sort(torch.zeros((tokens, choices), dtype=torch.int32, device=dev), 4)
    a = pca.int8_quant(torch.randn((tokens if gather else 0, 64), device=dev))
    b = pca.int8_quant(torch.randn((4, 48, 64), device=dev).transpose(1, 2), channel_axis=-1)
    assert pca.expert_bmm(a, b, plan, gather=gather).shape == (0, 48)
    assert pca.expert_bmm(a, b, plan, gather=gather, activation="swiglu").shape == (0, 24)


@pytest.mark.parametrize("tokens,choices", [(3, 0), (0, 2), (0, 0), (70, 0)])
def test_layers(dev, tokens, choices):
    layer = ExpertMLP(64, 32, 4, device=dev, dtype=torch.bfloat16)
    x = torch.randn((tokens, 64), device=dev).bfloat16()
    ids, w = torch.zeros((tokens, choices), dtype=torch.int64, device=dev), torch.rand((tokens, choices), device=dev)
    for form in (layer, layer.served()):
        with torch.no_grad():
            y = form(x, ids, w)
        assert torch.equal(y, torch.zeros_like(x))
