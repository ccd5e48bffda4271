"""Decode over fp8 caches whose scales are far from one.

Tolerances: those of test_gpu_latent.py for 16-bit operands, with what the two
operands of the second product may lose where they reach float16's subnormal
numbers (spacing 2^-24, so 2^-25 each). With S the largest scale of a group of
columns, an operand of values is code * 2^e with 2^e <= S < 2^(e + 1) and one of
weights p * scale / 2^e, so what the first loses counts up to twice, and what the
second loses up to S |code| times. A row's sum of weights is at least one (the
largest): the bound grows by 2^-25 (2 + S sum_t |code_t|)."""
from __future__ import annotations

import math

import pytest
import torch

import practice_cuda_amd as pca
from test_gpu_latent import BF16, F8, FP16, attend, near

pytestmark = pytest.mark.gpu


def check(dev, latent, rope, scale, ql, qr, softmax_scale, page=64, copies=1):
    """latent [n, dl] codes, rope [n, dr], scale [n, dl / 128], ql [heads, dl], qr [heads, dr]: one sequence, `copies` times."""
    n, dl = latent.shape
    dtype = ql.dtype
    pages = -(-n // page)
    g = torch.Generator(device=dev).manual_seed(n)
    order = torch.randperm(pages, generator=g, device=dev)
    cache = pca.LatentCache.empty(pages, page, latent_dim=dl, rope_dim=rope.shape[1], dtype=dtype, fp8=True, device=dev)
    at = order[torch.arange(n, device=dev) // page] * page + torch.arange(n, device=dev) % page
    cache.latent.view(torch.uint8).fill_(0x7F)  # NaN behind the last token
    cache.scale.fill_(math.nan)
    cache.rope.fill_(math.nan)
    cache.latent.view(torch.uint8).view(-1, dl)[at] = latent.view(torch.uint8)
    cache.scale.view(-1, dl // 128)[at] = scale
    cache.rope.view(-1, rope.shape[1])[at] = rope
    queries = (x.expand(copies, 1, *x.shape) for x in (ql, qr))
    out, lse = pca.latent_decode(*queries, cache, order.int().expand(copies, pages),
                                 torch.full((copies,), n, dtype=torch.int32, device=dev), softmax_scale=softmax_scale,
                                 return_lse=True)
    codes = latent.double()
    v = (codes.unflatten(-1, (-1, 128)) * scale.double().unsqueeze(-1)).flatten(1)
    limits = torch.full((ql.shape[0],), n, device=dev)
    want, want_lse, bound, bound_lse = attend(torch.cat([ql, qr], 1), torch.cat([v, rope.double()], 1), v, limits,
                                              softmax_scale, dtype)
    if dtype == FP16:
        top = scale.double().amax(0).repeat_interleave(128)
        bound = bound + 2.0 ** -25 * (2 + top * codes.abs().sum(0))
    near(out[:, 0], want, bound, "out")
    near(lse[:, 0], want_lse, bound_lse, "lse")


def tokens(dev, n, dl, dr, size, dtype, seed):
    """Codes and scales of N(0, size^2) latents, and rotary keys."""
    g = torch.Generator(device=dev).manual_seed(seed)
    q = pca.per_block_quant(size * torch.randn((n, dl), generator=g, device=dev), block_m=1, block_n=128, eps=1e-30)
    return g, q.tensor, torch.randn((n, dr), generator=g, device=dev).to(dtype), q.dequant_scale


@pytest.mark.parametrize("dl,dr", [(512, 64), (256, 32)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [5, 16, 30, 64, 128])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -10, 2.0 ** -4, 1.0, 2.0 ** 8, 2.0 ** 14])
def test_sizes_of_latents(dev, size, heads, dtype, dl, dr):
    g, codes, rope, scale = tokens(dev, 1500, dl, dr, size, dtype, heads)
    # scores of a few units whatever the size (float16 queries end at 65504 and at 2^-24)
    std = 0.1 / size
    share = 1.0 if std < 2.0 ** 12 and std > 2.0 ** -12 else 0.0
    ql = (share * std * torch.randn((heads, dl), generator=g, device=dev)).to(dtype)
    qr = torch.randn((heads, dr), generator=g, device=dev).to(dtype)
    check(dev, codes, rope, scale, ql, qr, 0.3)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dl,dr", [(512, 64), (256, 32)])
@pytest.mark.parametrize("size", [2.0 ** -10, 1.0, 2.0 ** 14])
def test_sizes_of_latents_of_many_sequences(dev, size, dtype, dl, dr):
    # more than 128 tiles: one workgroup takes 128 rows
    g, codes, rope, scale = tokens(dev, 300, dl, dr, size, dtype, 3)
    ql = torch.zeros((128, dl), device=dev).to(dtype)
    qr = torch.randn((128, dr), generator=g, device=dev).to(dtype)
    check(dev, codes, rope, scale, ql, qr, 0.3, copies=130)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,copies", [(16, 1), (64, 1), (128, 1), (16, 300), (64, 200), (128, 130)])
@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** -7, 1.0, 2.0 ** 8])
def test_peaked_head_over_a_long_tail(dev, size, heads, copies, dtype):
    """One token at the top and 65536 of them 12 below: the tail has 29 % of the weight. With many sequences a wave walks
    over all of one, or a quarter of it, and its weights all refer to the top token."""
    n, dl, dr = 65537, 512, 64
    g, codes, rope, scale = tokens(dev, n, dl, dr, size, dtype, heads)
    rope[:] = 0
    rope[n // 3, 0] = 12.0
    ql = torch.zeros((heads, dl), device=dev).to(dtype)
    qr = torch.zeros((heads, dr), device=dev).to(dtype)
    qr[:, 0] = 1.0
    # columns that do not average out
    codes = codes.float().abs().to(F8)
    check(dev, codes, rope, scale, ql, qr, 1.0, copies=copies)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [16, 128])
def test_scales_past_256(dev, dtype, heads):
    """Values that float16 does not hold, in an output that it does."""
    n, dl, dr = 5000, 512, 64
    g, codes, rope, scale = tokens(dev, n, dl, dr, 1.0, dtype, 7)
    scale = torch.empty_like(scale).uniform_(200.0, 2000.0, generator=g)
    ql = torch.zeros((heads, dl), device=dev).to(dtype)
    qr = torch.randn((heads, dr), generator=g, device=dev).to(dtype)
    assert (codes.float().abs().amax() * scale.amax()) > 65504
    check(dev, codes, rope, scale, ql, qr, 0.05)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [16, 64, 128])
def test_scales_of_many_sizes(dev, dtype, heads):
    """Scales between 2^-16 and 4, another in every token and group; tokens of zeros among them."""
    n, dl, dr = 3001, 512, 64
    g, codes, rope, scale = tokens(dev, n, dl, dr, 1.0, dtype, 9)
    scale = torch.exp2(torch.empty_like(scale).uniform_(-16.0, 2.0, generator=g))
    scale[::7] = 0.0
    scale[64:200] = 1e-12 / 448
    ql = (0.05 * torch.randn((heads, dl), generator=g, device=dev)).to(dtype)
    qr = torch.randn((heads, dr), generator=g, device=dev).to(dtype)
    check(dev, codes, rope, scale, ql, qr, 0.1)
