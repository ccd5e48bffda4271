"""The latent-attention layer where there is nothing yet: the first layer of a
stack, which has no residual."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd.latent_layer import LatentAttention

pytestmark = pytest.mark.gpu


def layer_of(dev):
    torch.manual_seed(0)
    return LatentAttention(256, 4, device=dev)


def test_first_layer(dev):
    """The input is normed as it is, and is the next residual."""
    layer = layer_of(dev)
    x = torch.randn((70, layer.hidden), device=dev).bfloat16()
    cache = pca.LatentCache.empty(3, 32, device=dev)
    at, cu = torch.arange(70, device=dev), torch.tensor([0, 70], dtype=torch.int32, device=dev)
    out, residual = layer.prefill(x, None, cache, at, at, cu)
    want, total = layer.prefill(x, torch.zeros_like(x), cache, at, at, cu)
    assert torch.equal(out, want) and torch.equal(residual, x) and torch.equal(total, x)
    table = torch.arange(3, dtype=torch.int32, device=dev)[None]
    args = (cache, at[:1] + 70, at[:1] + 70, table, torch.tensor([71], dtype=torch.int32, device=dev))
    out, residual = layer.decode(x[:1], None, *args)
    want, _ = layer.decode(x[:1], torch.zeros_like(x[:1]), *args)
    assert torch.equal(out, want) and torch.equal(residual, x[:1])
