"""Tokens that share a slot, as a padded batch's do: what that slot holds is not
defined, but every other slot is as without them, and each part of the shared one
is some token's."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared", [2, 300])
@pytest.mark.parametrize("fp8", [False, True])
def test_shared_slots(dev, fp8, shared):
    g = torch.Generator(device=dev).manual_seed(shared)
    n, page, pages = 500, 16, 40
    latent = torch.randn((n + shared, 512), generator=g, device=dev).bfloat16()
    rope = torch.randn((n + shared, 64), generator=g, device=dev).bfloat16()
    dummy = 77
    free = torch.arange(pages * page, device=dev)
    free = free[free != dummy]
    own = free[torch.randperm(free.numel(), generator=g, device=dev)[:n]]
    slots = torch.cat([own, torch.full((shared,), dummy, device=dev)])
    order = torch.randperm(n + shared, generator=g, device=dev)
    caches = []
    for keep in (order, order[order < n]):
        cache = pca.LatentCache.empty(pages, page, fp8=fp8, device=dev)
        for t in (cache.latent, cache.rope, cache.scale):
            if t is not None:
                t.view(torch.uint8).zero_()
        caches.append(pca.latent_append(cache, latent[keep], rope[keep], slots[keep]))
    parts = [[t.view(torch.uint8).view(pages * page, -1) for t in (c.latent, c.rope, c.scale) if t is not None]
             for c in caches]
    for with_them, without in zip(*parts):
        assert torch.equal(with_them[free], without[free])
    single = pca.LatentCache.empty(-(-shared // page), page, fp8=fp8, device=dev)
    pca.latent_append(single, latent[n:], rope[n:], torch.arange(shared, device=dev))
    for got, t in zip(parts[0], (t for t in (single.latent, single.rope, single.scale) if t is not None)):
        rows = t.view(torch.uint8).view(t.shape[0] * page, -1)[:shared]
        assert (rows == got[dummy]).any(0).all()
