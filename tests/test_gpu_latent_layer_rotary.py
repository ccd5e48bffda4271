"""Rotary positions of the latent-attention layer: their frequencies stay in 32
bits whatever type the layer's weights are moved to, and agree with the formula.

Tolerance: an angle is one fp32 product of a position (exact below 2^24) and a
frequency that is off by a few units in its last place: within 2^-21 of itself,
at positions of up to 40000 by 0.02; the rotated values are rounded to bfloat16
(2^-9 of a value, values of up to about 5)."""
from __future__ import annotations

import pytest
import torch

from practice_cuda_amd.latent_layer import LatentAttention

pytestmark = pytest.mark.gpu


def rotated(x, positions, base):
    half = x.shape[-1] // 2
    freq = base ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    angle = (positions.double()[:, None] * freq).view(x.shape[0], *(1,) * (x.ndim - 2), half)
    z = torch.complex(x[..., :half].double(), x[..., half:].double()) * torch.polar(torch.ones_like(angle), angle)
    return torch.cat([z.real, z.imag], -1)


@pytest.mark.parametrize("move", [None, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("base", [10000.0, 500.0])
def test_positions(dev, move, base):
    layer = LatentAttention(256, 3, rope_base=base, device=dev)
    if move is not None:
        layer.to(move)
        layer.to(torch.bfloat16)
    layer.cpu()
    layer.to(dev)
    assert layer.freq.dtype == torch.float32 and layer.freq.device == layer.w_out.device
    g = torch.Generator(device=dev).manual_seed(0)
    positions = torch.cat([torch.arange(100, device=dev), torch.randint(0, 40000, (900,), generator=g, device=dev)])
    for shape in ((1000, 64), (1000, 3, 64)):
        x = torch.randn(shape, generator=g, device=dev).bfloat16()
        got = layer._rotate(x, positions).double()
        want = rotated(x, positions, base)
        size = torch.hypot(*x.double().chunk(2, -1)).repeat(*(1,) * (x.ndim - 1), 2)
        bound = size * (2.0 ** -8 + 40000 * 2.0 ** -21)
        assert ((got - want).abs() <= bound).all()


def test_layer_moved_to_bfloat16(dev):
    torch.manual_seed(0)
    layer = LatentAttention(256, 3, device=dev)
    freq = layer.freq.clone()
    layer.to(torch.bfloat16)
    assert torch.equal(layer.freq, freq)
