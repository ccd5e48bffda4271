"""Prefill where scores are large in the kernel's own units: softmax scales of one
and more (queries scaled by the caller), beside rows that see no key and tiles
whose scores are all -inf. Tolerances: those of test_gpu_latent.py."""
from __future__ import annotations

import math

import pytest
import torch

import practice_cuda_amd as pca
from test_gpu_latent import BF16, FP16, attend, near, prefill_case

pytestmark = pytest.mark.gpu

# fewer keys than queries: the first rows of a wave see none, its last ones some
FEWER = [(50, 20), (33, 1), (200, 70), (300, 269), (7, 3), (40, 0), (64, 64)]


SPARE = [0, len(FEWER) * 8192]  # tiles of 128 rows, of 256


@pytest.mark.parametrize("spare", SPARE)
@pytest.mark.parametrize("widths", [(128, 64, 128), (64, 32, 64)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale", [1.0, 4.0, 64.0])
def test_rows_that_see_nothing(dev, scale, dtype, widths, spare):
    prefill_case(dev, FEWER, 2, dtype=dtype, widths=widths, scale=scale, seed=3, spare=spare, q_std=0.5 / scale)


@pytest.mark.parametrize("spare", SPARE)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_negative_scale(dev, dtype, spare):
    """A scale of -1 with the queries' signs turned is a scale of 1."""
    g = torch.Generator(device=dev).manual_seed(4)
    cu = torch.tensor([[0, 50, 83], [0, 20, 21]], dtype=torch.int32, device=dev)
    q = (0.5 * torch.randn((83 + spare, 3, 192), generator=g, device=dev)).to(dtype)
    k, v = (torch.randn((21, 3, 128), generator=g, device=dev).to(dtype) for _ in range(2))
    kr = torch.randn((21, 64), generator=g, device=dev).to(dtype)
    a, la = pca.latent_prefill(-q, k, kr, v, *cu, softmax_scale=-1.0, return_lse=True)
    b, lb = pca.latent_prefill(q, k, kr, v, *cu, softmax_scale=1.0, return_lse=True)
    assert torch.equal(a, b) and torch.equal(la, lb)
    for q0, n in ((0, 30), (50, 32), (83, spare)):  # see nothing
        assert (a[q0:q0 + n] == 0).all() and (la[q0:q0 + n] == -math.inf).all()
    assert torch.isfinite(la[30:50]).all() and torch.isfinite(la[82]).all()


@pytest.mark.parametrize("spare", [0, 8192])
@pytest.mark.parametrize("scale", [0.07, 1.0, 3.0])
@pytest.mark.parametrize("first", [1, 32, 40, 100])
def test_keys_of_minus_infinity(dev, first, scale, spare):
    """Keys that are -inf to every query take no part, also where they fill whole tiles."""
    n, heads = 130, 2
    g = torch.Generator(device=dev).manual_seed(first)
    q = (0.5 / scale * torch.randn((n + spare, heads, 192), generator=g, device=dev)).bfloat16()
    q[..., 128:] = 0.25
    k, v = (torch.randn((n, heads, 128), generator=g, device=dev).bfloat16() for _ in range(2))
    kr = torch.randn((n, 64), generator=g, device=dev).bfloat16()
    kr[:first] = -math.inf
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    out, lse = pca.latent_prefill(q, k, kr, v, cu, cu, softmax_scale=scale, return_lse=True)
    limits = torch.arange(n, device=dev) + 1 - first  # of the keys that are left
    for h in range(heads):
        key = torch.cat([k[first:, h], kr[first:]], 1)
        want, want_lse, bound, bound_lse = attend(q[:n, h], key, v[first:, h], limits, scale, BF16)
        near(out[:n, h], want, bound, f"out, head {h}")
        near(lse[:n, h], want_lse, bound_lse, f"lse, head {h}")
