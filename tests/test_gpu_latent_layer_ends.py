"""The latent-attention layer where there is nothing yet: the first layer of a
stack, which has no residual, and batches of no tokens."""
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


@pytest.mark.parametrize("widths", [(512, 64, 128), (256, 32, 64)])
@pytest.mark.parametrize("residual", [False, True])
def test_empty_batch(dev, residual, widths):
    latent, rope, head = widths
    layer = LatentAttention(256, 4, latent_dim=latent, rope_dim=rope, head_dim=head, device=dev)
    cache = pca.LatentCache.empty(3, 32, latent_dim=latent, rope_dim=rope, device=dev)
    x = torch.empty((0, layer.hidden), device=dev).bfloat16()
    none = torch.empty(0, dtype=torch.int64, device=dev)
    table, lens = torch.empty((0, 3), dtype=torch.int32, device=dev), torch.empty(0, dtype=torch.int32, device=dev)
    out, total = layer.decode(x, x if residual else None, cache, none, none, table, lens)
    assert out.shape == total.shape == (0, layer.hidden)
    for cu in ([0], [0, 0, 0]):
        cu = torch.tensor(cu, dtype=torch.int32, device=dev)
        out, total = layer.prefill(x, x if residual else None, cache, none, none, cu)
        assert out.shape == total.shape == (0, layer.hidden)
    # sequences without new tokens
    lens, table = torch.tensor([3, 1], dtype=torch.int32, device=dev), torch.zeros((2, 3), dtype=torch.int32, device=dev)
    out, total = layer.decode(x, x if residual else None, cache, none, none, table, lens)
    assert out.shape == total.shape == (0, layer.hidden)


def test_tokens_that_do_not_divide(dev):
    layer = layer_of(dev)
    cache = pca.LatentCache.empty(3, 32, device=dev)
    x = torch.zeros((3, layer.hidden), device=dev).bfloat16()
    at = torch.arange(3, device=dev)
    lens, table = torch.tensor([3, 1], dtype=torch.int32, device=dev), torch.zeros((2, 3), dtype=torch.int32, device=dev)
    before = cache.latent.zero_().clone()
    with pytest.raises(ValueError, match="3 tokens"):
        layer.decode(x, x, cache, at, at, table, lens)
    assert torch.equal(cache.latent, before)
