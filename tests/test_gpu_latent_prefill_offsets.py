"""Prefill offsets that do not start at the first row: rows ahead of the first
sequence belong to none, as those behind the last one do not."""
from __future__ import annotations

import math

import pytest
import torch

import practice_cuda_amd as pca

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences", [1, 5, 61, 62, 63, 64, 300])
@pytest.mark.parametrize("ahead", [1, 127, 128, 129, 300])
@pytest.mark.parametrize("spare", [0, 70])
def test_rows_ahead_of_the_first_sequence(dev, ahead, sequences, spare):
    g = torch.Generator(device=dev).manual_seed(ahead)
    lens = [(37 * i) % 50 + 1 for i in range(sequences)]
    n, heads = sum(lens), 3
    cu = torch.tensor([0] + lens, device=dev).cumsum(0).int()
    q = torch.randn((ahead + n + spare, heads, 192), generator=g, device=dev).bfloat16()
    k, v = (torch.randn((ahead + n, heads, 128), generator=g, device=dev).bfloat16() for _ in range(2))
    kr = torch.randn((ahead + n, 64), generator=g, device=dev).bfloat16()
    out = torch.full((ahead + n + spare, heads, 128), 7.0, device=dev).bfloat16()
    at = cu + ahead
    got, lse = pca.latent_prefill(q, k, kr, v, at, at, out=out, return_lse=True)
    want, want_lse = pca.latent_prefill(q[ahead:ahead + n], k[ahead:], kr[ahead:], v[ahead:], cu, cu, return_lse=True)
    assert torch.equal(got[ahead:ahead + n], want) and torch.equal(lse[ahead:ahead + n], want_lse)
    for part in (slice(0, ahead), slice(ahead + n, None)):
        assert (got[part] == 0).all() and (lse[part] == -math.inf).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("widths", [(128, 64, 128), (64, 32, 64)])
def test_rows_ahead_in_tiles_of_256_rows(dev, dtype, widths):
    # past 8192 rows a sequence
    dn, dr, dv = widths
    ahead, n, heads = 16500, 300, 2
    g = torch.Generator(device=dev).manual_seed(1)
    q = torch.randn((ahead + n, heads, dn + dr), generator=g, device=dev).to(dtype)
    k, v = (torch.randn((n, heads, w), generator=g, device=dev).to(dtype) for w in (dn, dv))
    kr = torch.randn((n, dr), generator=g, device=dev).to(dtype)
    cu_k = torch.tensor([0, n], dtype=torch.int32, device=dev)
    out = torch.full((ahead + n, heads, dv), 7.0, device=dev).to(dtype)
    got, lse = pca.latent_prefill(q, k, kr, v, cu_k + ahead, cu_k, out=out, return_lse=True)
    assert (got[:ahead] == 0).all() and (lse[:ahead] == -math.inf).all()
    want = pca.latent_prefill(q[ahead:], k, kr, v, cu_k, cu_k)
    torch.testing.assert_close(got[ahead:], want, rtol=2e-2, atol=2e-2)


def test_rows_of_no_sequence(dev):
    # a single offset past the first row: no sequence at all
    q = torch.ones((40, 2, 192), device=dev).bfloat16()
    k, kr = torch.ones((0, 2, 128), device=dev).bfloat16(), torch.ones((0, 64), device=dev).bfloat16()
    cu = torch.tensor([25], dtype=torch.int32, device=dev)
    out, lse = pca.latent_prefill(q, k, kr, k, cu, cu, out=torch.full((40, 2, 128), 7.0, device=dev).bfloat16(),
                                  return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
