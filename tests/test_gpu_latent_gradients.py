"""The norm and the latent-attention operators have no gradient: with inputs that
require one the results are as without, and going backward through them, or
writing into a caller's tensor, is an error instead of a missing gradient."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd.latent_layer import LatentAttention

pytestmark = pytest.mark.gpu


def data(dev, *shape):
    return torch.randn(shape, device=dev).bfloat16()


def calls(dev):
    """{name: (function of its tensors, their names and tensors)}."""
    cu = torch.tensor([0, 9], dtype=torch.int32, device=dev)
    cache = pca.LatentCache.empty(2, 16, device=dev)
    cache.latent.normal_()
    cache.rope.normal_()
    table, lens = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.tensor([9], dtype=torch.int32, device=dev)

    def norm(x, weight, residual):
        q, total = pca.rms_norm_quant(x, weight, residual=residual)
        return q.dequant_scale, total

    def decode(q_latent, q_rope):
        return pca.latent_decode(q_latent, q_rope, cache, table, lens, softmax_scale=0.1, return_lse=True)

    def prefill(q, k_nope, k_rope, v):
        return pca.latent_prefill(q, k_nope, k_rope, v, cu, cu, return_lse=True)

    return {
        "norm": (norm, {"x": data(dev, 9, 256), "weight": data(dev, 256), "residual": data(dev, 9, 256)}),
        "decode": (decode, {"q_latent": data(dev, 1, 1, 4, 512), "q_rope": data(dev, 1, 1, 4, 64)}),
        "prefill": (prefill, {"q": data(dev, 9, 2, 192), "k_nope": data(dev, 9, 2, 128), "k_rope": data(dev, 9, 64),
                              "v": data(dev, 9, 2, 128)}),
    }


CASES = [(f, t) for f, names in (("norm", ("x", "weight", "residual")), ("decode", ("q_latent", "q_rope")),
                                 ("prefill", ("q", "k_nope", "k_rope", "v"))) for t in names]


@pytest.mark.parametrize("name,which", CASES)
def test_backward_is_an_error(dev, name, which):
    fn, tensors = calls(dev)[name]
    want = fn(**tensors)
    assert not any(t.requires_grad for t in want)
    needs = {k: t.clone().requires_grad_(k == which) for k, t in tensors.items()}
    got = fn(**needs)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and a.requires_grad
        with pytest.raises(RuntimeError, match="no gradient"):
            a.float().sum().backward()
    with torch.no_grad():
        assert not any(t.requires_grad for t in fn(**needs))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(fn(**needs), want))


def test_codes_too(dev):
    x = data(dev, 4, 128).requires_grad_()
    q, total = pca.rms_norm_quant(x, torch.ones(128, device=dev))
    assert total is None and q.tensor.requires_grad
    with pytest.raises(RuntimeError, match="no gradient"):
        q.tensor.float().sum().backward()


def test_outputs_of_the_caller_are_refused(dev):
    x, w = data(dev, 4, 128).requires_grad_(), torch.ones(128, device=dev)
    held = torch.zeros((4, 128), device=dev).bfloat16()
    with pytest.raises(ValueError, match="requires? a gradient"):
        pca.rms_norm_quant(x, w, residual=held, residual_out=held)
    cache = pca.LatentCache.empty(2, 16, device=dev)
    cache.latent.zero_()
    table, lens = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.tensor([9], dtype=torch.int32, device=dev)
    ql, qr = data(dev, 1, 1, 4, 512).requires_grad_(), data(dev, 1, 1, 4, 64)
    with pytest.raises(ValueError, match="requires? a gradient"):
        pca.latent_decode(ql, qr, cache, table, lens, softmax_scale=0.1, out=torch.zeros_like(ql).detach())
    cu = torch.tensor([0, 9], dtype=torch.int32, device=dev)
    q, k, kr = data(dev, 9, 2, 192), data(dev, 9, 2, 128), data(dev, 9, 64)
    with pytest.raises(ValueError, match="requires? a gradient"):
        pca.latent_prefill(q, k, kr, k.clone().requires_grad_(), cu, cu, out=torch.zeros_like(k))
    slots = torch.arange(4, device=dev)
    for latent, rope, weight in ((data(dev, 4, 512).requires_grad_(), data(dev, 4, 64), None),
                                 (data(dev, 4, 512), data(dev, 4, 64).requires_grad_(), None),
                                 (data(dev, 4, 512), data(dev, 4, 64), torch.ones(512, device=dev).requires_grad_())):
        with pytest.raises(ValueError, match="requires? a gradient"):
            pca.latent_append(cache, latent, rope, slots, weight=weight)
        assert (cache.latent == 0).all()
        with torch.no_grad():
            pca.latent_append(cache, latent, rope, slots, weight=weight)
        assert (cache.latent[0, :4] != 0).any()
        cache.latent.zero_()
    assert (held == 0).all()


@pytest.mark.parametrize("which", ["x", "residual", "w_key"])
def test_layer(dev, which):
    layer = LatentAttention(256, 4, device=dev)
    x, r = data(dev, 9, 256), data(dev, 9, 256)
    cache = pca.LatentCache.empty(2, 16, device=dev)
    at, cu = torch.arange(9, device=dev), torch.tensor([0, 9], dtype=torch.int32, device=dev)
    table = torch.arange(2, dtype=torch.int32, device=dev)[None]
    lens = torch.tensor([10], dtype=torch.int32, device=dev)

    def both():
        return (*layer.prefill(x, r, cache, at, at, cu), *layer.decode(x[:1], r[:1], cache, at[:1] + 9, at[:1] + 9,
                                                                       table, lens))

    want = both()
    assert not any(t.requires_grad for t in want)
    {"x": x, "residual": r, "w_key": layer.w_key}[which].requires_grad_()
    for a, b in zip(both(), want):
        assert torch.equal(a, b) and a.requires_grad
        with pytest.raises(RuntimeError, match="no gradient"):
            a.float().sum().backward()
    with torch.no_grad():
        assert not any(t.requires_grad for t in both())
