"""Calls without a gradient refuse inputs with a forward-mode tangent, on the CPU (no kernel is launched on these
paths): such a tensor need not require a gradient, and its tangent would be left out of the result without a word."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import practice_cuda_amd as pca

BF16 = torch.bfloat16


def codes(*shape, axis):
    lies = shape if axis == -2 else (*shape[:-2], shape[-1], shape[-2])
    t = torch.zeros(lies, dtype=torch.int8)
    return pca.QuantResult(t if axis == -2 else t.transpose(-1, -2), torch.ones(lies[:-1]), "x", "channel",
                           {"channel_axis": axis})


def with_scale(q, scale):
    return pca.QuantResult(q.tensor, scale, q.impl, q.granularity, q.meta)


def calls():
    """(name, call of one of its inputs, that input)"""
    x, w = torch.zeros((4, 256), dtype=BF16), torch.ones(256, dtype=BF16)
    yield "int8_quant", lambda t: pca.int8_quant(t), x
    a, b, bias = codes(1, 4, 32, axis=-2), codes(1, 32, 6, axis=-1), torch.zeros(1, 4, 6)
    yield "int8_bmm", lambda t: pca.int8_bmm(with_scale(a, t), b), a.dequant_scale
    yield "int8_bmm", lambda t: pca.int8_bmm(a, with_scale(b, t)), b.dequant_scale
    yield "int8_bmm", lambda t: pca.int8_bmm(a, b, bias=t), bias
    plan = pca.ExpertPlan(torch.zeros(8, dtype=torch.int32), torch.zeros((4, 2), dtype=torch.int32),
                          torch.zeros(4, dtype=torch.int32))
    rows, experts = codes(8, 32, axis=-2), codes(3, 32, 6, axis=-1)
    yield "expert_bmm", lambda t: pca.expert_bmm(with_scale(rows, t), experts, plan), rows.dequant_scale
    yield "expert_bmm", lambda t: pca.expert_bmm(rows, with_scale(experts, t), plan), experts.dequant_scale
    yield "expert_bmm", lambda t: pca.expert_bmm(rows, experts, plan, bias=t), torch.zeros(3, 6)
    yield "rms_norm_quant", lambda t: pca.rms_norm_quant(t, w), x
    yield "rms_norm_quant", lambda t: pca.rms_norm_quant(x, t), w
    yield "rms_norm_quant", lambda t: pca.rms_norm_quant(x, w, residual=t), x
    cache, slots = pca.LatentCache.empty(4, 16, device="cpu"), torch.arange(3)
    latent, rope, norm = torch.zeros((3, 512), dtype=BF16), torch.zeros((3, 64), dtype=BF16), torch.ones(512)
    yield "latent_append", lambda t: pca.latent_append(cache, t, rope, slots), latent
    yield "latent_append", lambda t: pca.latent_append(cache, latent, t, slots), rope
    yield "latent_append", lambda t: pca.latent_append(cache, latent, rope, slots, weight=t), norm
    ql, qr = torch.zeros((2, 1, 16, 512), dtype=BF16), torch.zeros((2, 1, 16, 64), dtype=BF16)
    table, lens = torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    yield "latent_decode", lambda t: pca.latent_decode(t, qr, cache, table, lens, softmax_scale=0.1), ql
    yield "latent_decode", lambda t: pca.latent_decode(ql, t, cache, table, lens, softmax_scale=0.1), qr
    parts = [torch.zeros((5, 2, 192), dtype=BF16), torch.zeros((6, 2, 128), dtype=BF16),
             torch.zeros((6, 64), dtype=BF16), torch.zeros((6, 2, 128), dtype=BF16)]
    cu = torch.tensor([0, 5], dtype=torch.int32), torch.tensor([0, 6], dtype=torch.int32)
    for i in range(4):
        yield "latent_prefill", lambda t, i=i: pca.latent_prefill(*parts[:i], t, *parts[i + 1:], *cu), parts[i]


@pytest.mark.parametrize("name,call,value", [pytest.param(*c, id=f"{c[0]}-{i}") for i, c in enumerate(calls())])
def test_tangents_are_refused(name, call, value):
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(value, torch.ones_like(value))
        with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
            call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
            call(dual)
