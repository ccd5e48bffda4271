"""Prefill at the lengths that its tiles of 256 rows are for: a real sequence of
8192 queries and more, some of its rows and heads against 64 bits. Tolerances:
those of test_gpu_latent.py."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca
from test_gpu_latent import BF16, FP16, attend, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("queries,keys,heads", [(8192, 8192, 16), (8192, 9001, 16), (8333, 8333, 17), (16411, 16411, 8),
                                                (8200, 4000, 16), (20000, 300, 8)])
@pytest.mark.parametrize("widths", [(128, 64, 128), (64, 32, 64)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("causal", [True, False])
def test_long_sequence(dev, queries, keys, heads, widths, dtype, causal):
    assert queries * heads >= 8192 * 16
    dn, dr, dv = widths
    g = torch.Generator(device=dev).manual_seed(queries + keys)
    q = torch.randn((queries, heads, dn + dr), generator=g, device=dev).to(dtype)
    kv = torch.randn((keys, heads, dn + dv), generator=g, device=dev).to(dtype)
    kr = torch.randn((keys, dr), generator=g, device=dev).to(dtype)
    k, v = kv[..., :dn], kv[..., dn:]
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (queries, keys))
    scale = 2.0 * (dn + dr) ** -0.5
    out, lse = pca.latent_prefill(q, k, kr, v, cu_q, cu_k, softmax_scale=scale, causal=causal, return_lse=True)
    # the ends of tiles and of the sequence, and others between
    fixed = [0, 1, 31, 32, 255, 256, queries - keys, queries - keys + 1, queries // 2, queries - 257, queries - 256,
             queries - 129, queries - 128, queries - 2, queries - 1]
    rows = torch.tensor([r for r in fixed if 0 <= r], device=dev)
    rows = torch.cat([rows, torch.randint(0, queries, (185,), generator=g, device=dev)])
    limits = rows + (keys - queries + 1) if causal else torch.full_like(rows, keys)
    for h in (0, 1, heads // 2, heads - 1):
        key = torch.cat([k[:, h], kr], 1)
        want, want_lse, bound, bound_lse = attend(q[rows, h], key, v[:, h], limits, scale, dtype)
        near(out[rows, h], want, bound, f"out, head {h}")
        near(lse[rows, h], want_lse, bound_lse, f"lse, head {h}")
    assert torch.isfinite(out.float()).all()
