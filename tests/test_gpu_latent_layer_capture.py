"""The latent-attention layer where its weights' fp8 forms are made at a call: while
a graph is captured (nothing runs then), and on another stream than the next
call's."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd.latent_layer import LatentAttention

pytestmark = pytest.mark.gpu


def layer_of(dev, seed):
    torch.manual_seed(seed)
    return LatentAttention(256, 4, device=dev)


def inputs(dev):
    g = torch.Generator(device=dev).manual_seed(1)
    x, r = (torch.randn((70, 256), generator=g, device=dev).bfloat16() for _ in range(2))
    return x, r, torch.arange(70, device=dev), torch.tensor([0, 70], dtype=torch.int32, device=dev)


def prompt(layer, data, dev):
    x, r, at, cu = data
    return layer.prefill(x, r, pca.LatentCache.empty(3, 32, device=dev), at, at, cu)[0]


def warm(dev, data):
    """Everything loaded and allocated once, by another layer."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prompt(layer_of(dev, 9), data, dev)
    torch.cuda.synchronize()


@pytest.mark.parametrize("stale", [False, True])
def test_capture_before_the_first_call(dev, stale):
    """stale: the layer has codes, of weights that changed since."""
    data, other = inputs(dev), layer_of(dev, 5)
    warm(dev, data)
    want = prompt(other, data, dev).clone()
    layer = layer_of(dev, 5 if not stale else 0)
    if stale:
        assert not torch.equal(prompt(layer, data, dev), want)
        layer.load_state_dict(other.state_dict())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = prompt(layer, data, dev)
    assert torch.equal(prompt(layer, data, dev), want)  # ahead of any replay
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
        assert torch.equal(prompt(layer, data, dev), want)
    del graph, held
    torch.cuda.empty_cache()
    filler = torch.full((64 << 20,), 0x55, dtype=torch.uint8, device=dev)  # takes what the graph gave back
    assert torch.equal(prompt(layer, data, dev), want)
    del filler


@pytest.mark.parametrize("call", ["quantize", "prefill"])
def test_codes_made_on_another_stream(dev, call):
    data, other = inputs(dev), layer_of(dev, 5)
    warm(dev, data)
    want = prompt(other, data, dev).clone()
    layer = layer_of(dev, 5)
    a = torch.randn((8192, 8192), device=dev).bfloat16()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(10):
            a @ a  # milliseconds ahead of the codes
        layer.quantize() if call == "quantize" else prompt(layer, data, dev)
    got = prompt(layer, data, dev)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
