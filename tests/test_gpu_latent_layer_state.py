"""The latent-attention layer's weights after they have changed: its fp8 forms follow."""
from __future__ import annotations

import copy

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd.latent_layer import LatentAttention

pytestmark = pytest.mark.gpu

NAMES = ("w_query", "w_latent", "w_key", "w_value", "w_out")


def layer_of(dev, seed=0, hidden=256, heads=4):
    torch.manual_seed(seed)
    return LatentAttention(hidden, heads, device=dev)


def prompt(layer, dev, n=70, residual=True):
    g = torch.Generator(device=dev).manual_seed(1)
    x, r = (torch.randn((n, layer.hidden), generator=g, device=dev).bfloat16() for _ in range(2))
    cache = pca.LatentCache.empty(3, 32, device=dev)
    at = torch.arange(n, device=dev)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    return layer.prefill(x, r if residual else None, cache, at, at, cu)


def changes(dev):
    other = layer_of(dev, 5)

    def load(layer):
        layer.load_state_dict(other.state_dict())

    def assign(layer):
        layer.load_state_dict(copy.deepcopy(other.state_dict()), assign=True)

    def in_place(layer):
        with torch.no_grad():
            for name in NAMES:
                getattr(layer, name).copy_(getattr(other, name))

    def in_inference_mode(layer):
        with torch.inference_mode():
            for name in NAMES:
                getattr(layer, name).copy_(getattr(other, name))

    def replace(layer):
        for name in NAMES:
            setattr(layer, name, torch.nn.Parameter(getattr(other, name).clone(), requires_grad=False))

    def through_the_cpu(layer):
        layer.cpu()
        with torch.no_grad():
            for name in NAMES:
                getattr(layer, name).copy_(getattr(other, name))
        layer.to(dev)

    return other, {f.__name__: f for f in (load, assign, in_place, in_inference_mode, replace, through_the_cpu)}


@pytest.mark.parametrize("how", ["load", "assign", "in_place", "in_inference_mode", "replace", "through_the_cpu"])
@pytest.mark.parametrize("quantized", [False, True])  # by a call of quantize(), or by use
def test_changed_weights_are_used(dev, how, quantized):
    other, ways = changes(dev)
    want, _ = prompt(other, dev)
    layer = layer_of(dev, 0)
    if quantized:
        layer.quantize()
    before, _ = prompt(layer, dev)
    assert not torch.equal(before, want)
    ways[how](layer)
    got, _ = prompt(layer, dev)
    assert torch.equal(got, want)


def test_codes_made_in_inference_mode(dev):
    layer, other = layer_of(dev, 0), layer_of(dev, 5)
    with torch.inference_mode():
        prompt(layer, dev)
    layer.load_state_dict(other.state_dict())
    got, _ = prompt(layer, dev)
    want, _ = prompt(other, dev)
    assert torch.equal(got, want)


def test_other_shapes_and_types(dev):
    """Codes of weights that no longer fit are made anew."""
    layer, other = layer_of(dev, 0).quantize(), layer_of(dev, 5, hidden=384)
    layer.hidden = 384
    for name in ("norm", *NAMES):
        setattr(layer, name, torch.nn.Parameter(getattr(other, name).clone(), requires_grad=False))
    got, _ = prompt(layer, dev)
    want, _ = prompt(other, dev)
    assert torch.equal(got, want)
    layer.half()  # weights of another type and back: two roundings
    layer.bfloat16()
    other.half()
    other.bfloat16()
    got, _ = prompt(layer, dev)
    want, _ = prompt(other, dev)
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", NAMES)
def test_each_weight_is_watched(dev, name):
    layer = layer_of(dev)
    before, _ = prompt(layer, dev)
    with torch.no_grad():
        getattr(layer, name).mul_(-0.5)
    after, _ = prompt(layer, dev)
    assert not torch.equal(before, after)


def test_unchanged_weights_are_quantized_once(dev):
    layer = layer_of(dev).quantize()
    codes = layer._fp8
    prompt(layer, dev)
    prompt(layer, dev)
    assert layer._fp8 is codes


def test_copies_and_inference_tensors(dev):
    layer = layer_of(dev)
    want, _ = prompt(layer, dev)
    twin = copy.deepcopy(layer)
    with torch.no_grad():
        layer.w_out.zero_()
    got, _ = prompt(twin, dev)
    assert torch.equal(got, want)
    with torch.inference_mode():
        layer = layer_of(dev)
        got, _ = prompt(layer, dev)
        assert torch.equal(got, want)


def test_a_captured_step_follows_its_weights(dev):
    """The codes stay where they are, so that a graph reads the new ones after quantize()."""
    layer, other = layer_of(dev, 0).quantize(), layer_of(dev, 5)
    g = torch.Generator(device=dev).manual_seed(2)
    x, r = (torch.randn((2, layer.hidden), generator=g, device=dev).bfloat16() for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    lens, places = torch.tensor([1, 1], dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    slots = torch.tensor([0, 64], device=dev)

    def step(layer, cache):
        return layer.decode(x, r, cache, slots, places, table, lens)[0]

    cache = pca.LatentCache.empty(4, 32, device=dev)
    before = step(layer, cache).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(layer, cache)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, before)
    layer.load_state_dict(other.state_dict())
    layer.quantize()
    want = step(other, pca.LatentCache.empty(4, 32, device=dev)).clone()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
    assert not torch.equal(before, want)
