"""expert_sort, expert_dispatch, expert_combine and expert_bmm on the GPU against
their definitions in 64 bits, their gradients against the formulas and against
differences, and a run of them together."""
from __future__ import annotations

import math

import pytest
import torch

import practice_cuda_amd as pca
from practice_cuda_amd.expert_layer import ExpertMLP, Int8Experts
from practice_cuda_amd.modules import convert_to_float8_bmm_training

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def sorted_by(ids, experts):
    """order, place and starts as lists, from the definition."""
    flat = ids.flatten().tolist()
    groups = [[p for p, e in enumerate(flat) if e == g] for g in range(experts)] if experts <= 16 else None
    if groups is None:
        groups = [[] for _ in range(experts)]
        for p, e in enumerate(flat):
            if 0 <= e < experts:
                groups[e].append(p)
    none = [p for p, e in enumerate(flat) if not 0 <= e < experts]
    order, starts, place = [], [0], [0] * len(flat)
    for group in groups:
        order += group
        starts.append(len(order))
    for s, p in enumerate(order):
        place[p] = s
    for p in none:
        place[p] = -1 - len(order)
        order.append(p)
    return order, place, starts


def check_sort(ids, experts):
    plan = pca.expert_sort(ids, experts)
    order, place, starts = sorted_by(ids, experts)
    assert plan.order.tolist() == order
    assert plan.place.flatten().tolist() == place and plan.place.shape == ids.shape
    assert plan.starts.tolist() == starts and plan.experts == experts
    return plan


def ids_of(dev, tokens, choices, experts, seed=0, dtype=torch.int32, none=0.1):
    g = torch.Generator(device=dev).manual_seed(seed + tokens)
    ids = torch.randint(0, experts, (tokens, choices), generator=g, device=dev)
    ids[torch.rand(ids.shape, generator=g, device=dev) < none] = -1
    return ids.to(dtype)


@pytest.mark.parametrize("tokens,choices,experts", [
    (1, 1, 1), (1, 8, 256), (5, 3, 2), (64, 1, 7), (63, 8, 64), (512, 8, 1024), (513, 8, 1023), (1000, 4, 3),
    (4096, 1, 16), (4097, 1, 16), (2049, 2, 60), (9000, 8, 128), (40000, 6, 1024), (70001, 2, 5)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort(dev, tokens, choices, experts, dtype):
    check_sort(ids_of(dev, tokens, choices, experts, dtype=dtype), experts)


def test_sort_extremes(dev):
    for tokens in (300, 9000):
        for value in (0, 6, -1, 7, 2**31 - 1):
            check_sort(torch.full((tokens, 2), value, dtype=torch.int32, device=dev), 7)
    check_sort(torch.tensor([[2**40, 1], [-2**40, 0]], device=dev), 2)  # ids past 32 bits are no expert's
    for shape in ((0, 4), (5, 0)):
        plan = pca.expert_sort(torch.zeros(shape, dtype=torch.int32, device=dev), 9)
        assert plan.starts.tolist() == [0] * 10 and plan.order.numel() == 0 and plan.place.shape == shape
    check_sort(torch.arange(512, device=dev).flip(0).reshape(64, 8).int() % 64, 64)
    check_sort(ids_of(dev, 50, 128, 9), 9)


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------
WIDTHS = [1, 7, 8, 64, 1000, 1031, 4096, 7168]


def half(t):
    return torch.finfo(t).eps / 2


def rounded(t, v):
    """Half a step of type t at v. Below the smallest normal number the steps stay those at it (fp16: 2^-24, so half
    a step is 2^-25 = 2^-11 * 2^-14), so that is where the relative form ends."""
    return half(t) * v.abs().clamp(min=torch.finfo(t).smallest_normal)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("tokens,choices", [(1, 1), (3, 8), (130, 4)])
def test_dispatch(dev, tokens, choices, width, dtype):
    ids = ids_of(dev, tokens, choices, 6)
    plan = pca.expert_sort(ids, 6)
    x = torch.randn((tokens, width), device=dev).to(dtype).requires_grad_()
    out = pca.expert_dispatch(x, plan)
    used = plan.starts[-1].item()
    assert torch.equal(out[:used], x.detach()[plan.order[:used].long() // choices])
    assert not out[used:].any()
    assert torch.equal(pca.expert_dispatch(x.detach(), plan), out)
    g = torch.randn(out.shape, device=dev).to(dtype)
    back, = torch.autograd.grad(out, x, g)
    parts = g.double()[plan.place.clamp(min=0).long()] * (plan.place >= 0).unsqueeze(-1)
    want, size = parts.sum(1), parts.abs().sum(1)
    # up to `choices` additions in fp32, one rounding
    assert ((back.double() - want).abs() <= rounded(dtype, want) + (choices + 1) * U * size).all()


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,w_dtype", [(BF16, FP32), (FP16, FP32), (FP32, FP32), (BF16, BF16), (FP32, FP16)])
@pytest.mark.parametrize("tokens,choices", [(1, 1), (3, 8), (130, 4)])
def test_combine(dev, tokens, choices, width, dtype, w_dtype):
    plan = pca.expert_sort(ids_of(dev, tokens, choices, 6), 6)
    rows = torch.randn((tokens * choices, width), device=dev).to(dtype)
    rows[plan.starts[-1].item():] = math.nan  # what pairs without an expert hold is never used
    rows.requires_grad_()
    w = torch.rand((tokens, choices), device=dev).to(w_dtype).requires_grad_()
    out = pca.expert_combine(rows, plan, w)
    assert torch.equal(pca.expert_combine(rows.detach(), plan, w.detach()), out)
    used = (plan.place >= 0).unsqueeze(-1)
    y = torch.where(used, rows.detach().double()[plan.place.clamp(min=0).long()], 0.0)
    parts = y * w.detach().double().unsqueeze(-1)
    want, size = parts.sum(1), parts.abs().sum(1)
    assert ((out.double() - want).abs() <= rounded(dtype, want) + (choices + 2) * U * size).all()
    g = torch.randn(out.shape, device=dev).to(dtype)
    to_rows, to_weights = torch.autograd.grad(out, (rows, w), g)
    want = torch.zeros((tokens * choices, width), dtype=torch.float64, device=dev)
    flat = plan.place.flatten()
    sel = flat >= 0
    want[flat[sel].long()] = (g.double().unsqueeze(1) * w.detach().double().unsqueeze(-1)).flatten(0, 1)[sel]
    assert ((to_rows.double() - want).abs() <= rounded(dtype, want) + U * want.abs()).all()
    dots = (y * g.double().unsqueeze(1)).sum(-1)
    size = (y * g.double().unsqueeze(1)).abs().sum(-1)
    # a sum of `width` products: at most one rounding a product and one an addition on the way of each
    assert to_weights.dtype == w_dtype
    steps = 2 + min(width, 8) + math.ceil(width / 2048) + 6 + 4
    err = rounded(w_dtype, dots) if w_dtype != FP32 else 0.0
    assert ((to_weights.double() - dots).abs() <= err + steps * U * size).all()


def test_one_gradient_at_a_time(dev):
    plan = pca.expert_sort(ids_of(dev, 40, 3, 5), 5)
    rows, w = torch.randn((120, 48), device=dev), torch.rand((40, 3), device=dev)
    g = torch.randn((40, 48), device=dev)
    a, b = rows.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(pca.expert_combine(a, plan, b), (a, b), g)
    assert torch.equal(torch.autograd.grad(pca.expert_combine(a, plan, w), a, g)[0], both[0])
    assert torch.equal(torch.autograd.grad(pca.expert_combine(rows, plan, b), b, g)[0], both[1])


def test_gradients_against_differences(dev):
    """Both are linear in rows, weights and tokens, so a central difference of any step is exact but for rounding:
    fp32 sums of 24 values up to about 10, over a step of one."""
    plan = pca.expert_sort(ids_of(dev, 4, 2, 3), 3)
    x = torch.randn((4, 6), device=dev)
    w = torch.rand((4, 2), device=dev)
    c = torch.randn((4, 6), device=dev)
    scale = torch.randn((8, 1), device=dev)

    def f(x, w):
        return (pca.expert_combine(pca.expert_dispatch(x, plan) * scale, plan, w) * c).sum()

    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(f(xs, ws), (xs, ws))
    for t, grad, of in ((x, gx, lambda v: f(v, w)), (w, gw, lambda v: f(x, v))):
        for i in range(t.numel()):
            step = torch.zeros_like(t).flatten()
            step[i] = 0.5
            diff = of(t + step.view(t.shape)) - of(t - step.view(t.shape))
            assert abs(diff.item() - grad.flatten()[i].item()) < 1e-4


def test_row_views(dev):
    """Strided rows, broadcast tokens and gradients, rows that 16 bytes do not divide."""
    plan = pca.expert_sort(ids_of(dev, 30, 2, 4), 4)
    wide = torch.randn((30, 300), device=dev).to(BF16)
    for x in (wide[:, 8:264], wide[:, 3:100], wide[:1, :64].expand(30, 64), wide[:, :1]):
        assert torch.equal(pca.expert_dispatch(x, plan), pca.expert_dispatch(x.contiguous(), plan))
    rows = torch.randn((60, 300), device=dev).to(BF16)
    w = torch.rand((30, 2), device=dev)
    for r in (rows[:, 8:264], rows[:, 5:100], rows[:1].expand(60, 300)):
        assert torch.equal(pca.expert_combine(r, plan, w), pca.expert_combine(r.contiguous(), plan, w))
    x = wide[:1, :64].clone().requires_grad_()
    pca.expert_dispatch(x.expand(30, 64), plan).float().sum().backward()  # a broadcast input and a broadcast gradient
    used = plan.starts[-1].item()
    assert torch.equal(x.grad, torch.full_like(x, used))
    r = rows.clone().requires_grad_()
    pca.expert_combine(r, plan, w).float().sum().backward()
    assert torch.equal(r.grad[plan.place[0, 0].item()] if plan.place[0, 0] >= 0 else r.grad[0] * 0,
                       (w[0, 0].to(BF16) * torch.ones(300, device=dev, dtype=BF16)) if plan.place[0, 0] >= 0 else r.grad[0] * 0)


def test_no_tokens(dev):
    plan = pca.expert_sort(torch.zeros((0, 2), dtype=torch.int32, device=dev), 4)
    assert pca.expert_dispatch(torch.zeros((0, 8), device=dev), plan).shape == (0, 8)
    assert pca.expert_combine(torch.zeros((0, 8), device=dev), plan, torch.zeros((0, 2), device=dev)).shape == (0, 8)
    plan = pca.expert_sort(torch.zeros((3, 0), dtype=torch.int32, device=dev), 4)
    out = pca.expert_combine(torch.zeros((0, 8), device=dev), plan, torch.zeros((3, 0), device=dev))
    assert torch.equal(out, torch.zeros((3, 8), device=dev))  # a sum over no choices
    x = torch.ones((3, 8), device=dev, requires_grad=True)
    pca.expert_dispatch(x, plan).sum().backward()
    assert torch.equal(x.grad, torch.zeros_like(x))


# ---------------------------------------------------------------------------
# the experts' products
# ---------------------------------------------------------------------------
def codes(g, shape):
    wide = -(-shape[-1] // 16) * 16
    t = torch.randint(-128, 128, (*shape[:-1], wide), generator=g, device=g.device, dtype=torch.int8)[..., :shape[-1]]
    return t, torch.rand(shape[:-1], generator=g, device=g.device) + 0.5


def run(dev, tokens, choices, experts, n, k, *, gather, ids=None, out=BF16, activation="none", bias=False, seed=0):
    g = torch.Generator(device=dev).manual_seed(tokens + 10 * n + k + seed)
    ids = ids_of(dev, tokens, choices, experts, seed) if ids is None else ids
    plan = pca.expert_sort(ids, experts)
    pairs = tokens * choices
    a, sa = codes(g, (tokens if gather else pairs, k))
    sa = sa / (74.0 * 74.0 * math.sqrt(max(k, 1)))
    w, sw = codes(g, (experts, n, k))
    bias = torch.randn((experts, n), generator=g, device=dev).to(FP16) if bias else None
    y = pca.expert_bmm(pca.QuantResult(a, sa, "x", "channel", {"channel_axis": -2}),
                       pca.QuantResult(w.transpose(1, 2), sw, "x", "channel", {"channel_axis": -1}), plan,
                       gather=gather, out_dtype=out, bias=bias, activation=activation)
    starts = plan.starts.tolist()
    assert y.shape == (pairs, n // 2 if activation == "swiglu" else n) and y.dtype == out
    assert not y[starts[-1]:].any()
    rows = plan.order.long() // choices if gather else torch.arange(pairs, device=dev)
    for e in range(experts):
        lo, hi = starts[e], starts[e + 1]
        if hi == lo:
            continue
        at = rows[lo:hi]
        v = torch.matmul(a[at].double(), w[e].double().t().contiguous()) * (sa[at].double()[:, None] * sw[e].double())
        d = 3.01 * U * v.abs()
        if bias is not None:
            v = v + bias[e].double()
            d = d + 1.01 * U * (v.abs() + d)
        if activation == "gelu":
            v, d = 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5))), 1.13 * d + 8 * U * v.abs()
        elif activation == "swiglu":
            h = n // 2
            s = v[:, :h] * torch.sigmoid(v[:, :h])
            ds = 1.1 * d[:, :h] + 16 * U * s.abs()
            up, du = v[:, h:], d[:, h:]
            v, d = s * up, ds * up.abs() + s.abs() * du + ds * du + 2 * U * (s * up).abs()
        tiny = torch.finfo(out).smallest_normal
        assert ((y[lo:hi].double() - v).abs() <= 1.01 * d + half(out) * (v.abs() + d).clamp(min=tiny)).all(), f"expert {e}"
    return y


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("tokens,choices,experts,n,k", [
    (1, 1, 1, 16, 64), (1, 2, 4, 70, 100), (24, 8, 64, 96, 256), (7, 3, 200, 33, 1031), (100, 2, 3, 130, 272),
    (300, 4, 8, 200, 384), (1000, 2, 5, 258, 512), (700, 6, 60, 64, 128), (2500, 2, 4, 320, 640)])
def test_expert_bmm(dev, tokens, choices, experts, n, k, gather):
    run(dev, tokens, choices, experts, n, k, gather=gather)


@pytest.mark.parametrize("out", [BF16, FP16, FP32])
@pytest.mark.parametrize("activation", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("tokens", [20, 900])
def test_expert_bmm_epilogue(dev, tokens, bias, activation, out):
    run(dev, tokens, 3, 6, 258, 400, gather=True, out=out, activation=activation, bias=bias)


def test_expert_bmm_uneven(dev):
    """All rows at one expert, at the last one, at none; groups whose sizes end next to the tiles' ends."""
    for tokens in (40, 1200):
        for value in (0, 5, -1):
            run(dev, tokens, 2, 6, 96, 192, gather=True, ids=torch.full((tokens, 2), value, dtype=torch.int32, device=dev))
    sizes = [0, 1, 15, 16, 17, 0, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 0, 2, 383]
    ids = torch.repeat_interleave(torch.arange(len(sizes), device=dev), torch.tensor(sizes, device=dev))
    ids = ids[torch.randperm(ids.numel(), device=dev)].int()[:, None].contiguous()
    for gather in (False, True):
        run(dev, ids.shape[0], 1, len(sizes), 160, 320, gather=gather, ids=ids)
    few = torch.tensor([[0, 2], [5, 2]], dtype=torch.int32, device=dev)
    run(dev, 2, 2, 6, 64, 64, gather=True, ids=few)
    run(dev, 2, 2, 6, 64, 64, gather=True, ids=torch.zeros_like(few))  # a token twice at one expert


@pytest.mark.parametrize("k", [1, 16, 17, 127, 129, 300])
def test_expert_bmm_inner(dev, k):
    for tokens in (10, 800):
        run(dev, tokens, 2, 4, 100, k, gather=True, out=FP32)


def test_expert_bmm_output(dev):
    """A given output with guards around it, and one matrix for every expert."""
    g = torch.Generator(device=dev).manual_seed(2)
    plan = pca.expert_sort(ids_of(dev, 30, 2, 4), 4)
    a, sa = codes(g, (60, 96))
    w, sw = codes(g, (1, 72, 96))
    qa = pca.QuantResult(a, sa, "x", "channel", {"channel_axis": -2})
    qb = pca.QuantResult(w.expand(4, -1, -1).transpose(1, 2), sw.expand(4, -1), "x", "channel", {"channel_axis": -1})
    want = pca.expert_bmm(qa, qb, plan)
    wide = torch.full((62, 80), 7.0, dtype=BF16, device=dev)
    assert torch.equal(pca.expert_bmm(qa, qb, plan, out=wide[1:61, 5:77]), want)
    wide[1:61, 5:77] = 7.0
    assert (wide == 7.0).all()
    with pytest.raises(ValueError, match="16-byte aligned"):
        pca.expert_bmm(pca.QuantResult(torch.zeros((60, 104), dtype=torch.int8, device=dev)[:, 8:], sa, "x", "channel",
                                       qa.meta), qb, plan)


def test_plans_that_are_none(dev):
    """Places, orders and starts past what they index read and write nothing else's memory."""
    ids = ids_of(dev, 40, 2, 4, none=0.0)
    good = pca.expert_sort(ids, 4)
    bad = pca.ExpertPlan(good.order + 1000, good.place + 70, good.starts * 3)
    x = torch.ones((40, 64), device=dev)
    pca.expert_dispatch(x, bad)
    pca.expert_combine(torch.ones((80, 64), device=dev), bad, torch.ones((40, 2), device=dev))
    g = torch.Generator(device=dev).manual_seed(1)
    a, sa = codes(g, (40, 64))
    w, sw = codes(g, (4, 32, 64))
    for plan in (bad, pca.ExpertPlan(-good.order, good.place, good.starts.flip(0).contiguous())):
        pca.expert_bmm(pca.QuantResult(a, sa, "x", "channel", {"channel_axis": -2}),
                       pca.QuantResult(w.transpose(1, 2), sw, "x", "channel", {"channel_axis": -1}), plan, gather=True)
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def plain_experts(x, ids, weights, gate_up, down):
    """The layer in 64 bits."""
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for t in range(ids.shape[0]):
        for j in range(ids.shape[1]):
            e = ids[t, j].item()
            if 0 <= e < down.shape[0]:
                gate, up = (gate_up[e].double() @ x[t].double()).chunk(2)
                y[t] = y[t] + weights[t, j].double() * (down[e].double() @ (gate * torch.sigmoid(gate) * up))
    return y


def test_layer_and_served_form(dev):
    """Served outputs against the formula with the layer's own roundings: codes of weights, tokens and inner rows.

    The quantizers' steps are half of 1/127 of a row's largest value; their effect on an output is a sum of
    independent errors, bounded here by their root of squares times 6."""
    torch.manual_seed(4)
    layer = ExpertMLP(64, 48, 5, device=dev, dtype=BF16)
    x = torch.randn((37, 64), device=dev).to(BF16)
    ids = ids_of(dev, 37, 2, 5)
    w = torch.rand((37, 2), device=dev)
    gate_up = torch.cat([m.weight for m in layer.gate_up]).detach()
    down = torch.cat([m.weight for m in layer.down]).detach()
    served = layer.served()
    assert isinstance(served, Int8Experts)
    y = served(x, ids, w)
    # the same with dequantized operands, in 64 bits: what is left are bf16 roundings of the inner rows, of both
    # products and of the sum, and the inner rows' codes
    deq = [q.double() * s.double().unsqueeze(-1) for q, s in ((served.gate_up, served.gate_up_scale),
                                                             (served.down, served.down_scale))]
    q = pca.int8_quant(x)
    xq = q.tensor.double() * q.dequant_scale.double().unsqueeze(-1)
    want = torch.zeros((37, 64), dtype=torch.float64, device=dev)
    room = torch.zeros_like(want)
    for t in range(37):
        for j in range(2):
            e = ids[t, j].item()
            if e < 0:
                continue
            gate, up = (deq[0][e] @ xq[t]).chunk(2)
            h = gate * torch.sigmoid(gate) * up
            step = 2.0 ** -8 * h.abs() + h.abs().max() * (1 + 2.0 ** -8) / 254 + 1e-5 * h.abs().max()
            out = deq[1][e] @ h
            d = deq[1][e].abs() @ step
            want[t] += w[t, j].double() * out
            room[t] += w[t, j].double() * (d + 2.0 ** -8 * (out.abs() + d))
    assert ((y.double() - want).abs() <= 1.01 * room + 2.0 ** -8 * (want.abs() + room)).all()
    # and the layer itself in bf16 is near the formula: three products' roundings
    out = layer(x, ids, w)
    ref = plain_experts(x, ids, w, gate_up, down)
    assert (out.double() - ref).norm() <= 0.02 * ref.norm()
    assert (y.double() - ref).norm() <= 0.05 * ref.norm()
    with pytest.raises(RuntimeError, match="no gradient"):
        served(x.clone().requires_grad_(), ids, w).sum().backward()


def test_layer_gradients(dev):
    """In fp32 against the formula's own gradients in 64 bits; all sums are shorter than 400."""
    torch.manual_seed(5)
    layer = ExpertMLP(32, 24, 4, device=dev, dtype=FP32)
    x = torch.randn((50, 32), device=dev, requires_grad=True)
    ids = ids_of(dev, 50, 3, 4)
    w = torch.rand((50, 3), device=dev, requires_grad=True)
    c = torch.randn((50, 32), device=dev)
    params = [m.weight for m in layer.gate_up] + [m.weight for m in layer.down]
    got = torch.autograd.grad((layer(x, ids, w) * c).sum(), [x, w, *params])
    x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    p64 = [p.detach().double().requires_grad_() for p in params]
    y = plain_experts(x64, ids, w64, torch.cat(p64[:4]), torch.cat(p64[4:]))
    want = torch.autograd.grad((y * c.double()).sum(), [x64, w64, *p64])
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 1e-5 * b.norm()


def test_fp8_layer_trains(dev):
    """The converted layer runs forward and backward, with gradients near those of the bf16 layer (fp8 steps of 2^-4
    in each operand of three products)."""
    torch.manual_seed(6)
    layer = ExpertMLP(128, 128, 3, device=dev, dtype=BF16)
    x = torch.randn((300, 128), device=dev).to(BF16).requires_grad_()
    ids = ids_of(dev, 300, 2, 3)
    w = torch.rand((300, 2), device=dev, requires_grad=True)
    params = [m.weight for m in layer.gate_up] + [m.weight for m in layer.down]
    want = torch.autograd.grad(layer(x, ids, w).float().sum(), [x, w, *params])
    convert_to_float8_bmm_training(layer)
    got = torch.autograd.grad(layer(x, ids, w).float().sum(), [x, w, *params])
    for a, b in zip(got, want):
        assert a.shape == b.shape and (a.double() - b.double()).norm() <= 0.2 * b.double().norm()


def test_served_state(dev):
    torch.manual_seed(7)
    layer = ExpertMLP(64, 32, 3, device=dev, dtype=BF16)
    served = layer.served()
    x, ids, w = torch.randn((9, 64), device=dev).to(BF16), ids_of(dev, 9, 2, 3), torch.rand((9, 2), device=dev)
    want = served(x, ids, w)
    assert torch.equal(served.to(BF16)(x, ids, w), want) and served.down_scale.dtype == FP32
    other = ExpertMLP(64, 32, 3, device=dev, dtype=BF16).served()
    other.load_state_dict(served.state_dict())
    assert torch.equal(other(x, ids, w), want)
    with pytest.raises(ValueError, match="multiples of 16"):
        Int8Experts(torch.zeros((2, 24, 32), device=dev), torch.zeros((2, 32, 12), device=dev))
    with pytest.raises(ValueError, match="gate_up must be"):
        Int8Experts(torch.zeros((2, 24, 32), device=dev), torch.zeros((2, 32, 16), device=dev))


def test_served_graph(dev):
    """One captured graph serves any routing; eager work runs between the replays."""
    torch.manual_seed(8)
    served = ExpertMLP(128, 64, 8, device=dev, dtype=BF16).served()
    for tokens in (5, 3000):  # one launch and two of the sort; both kinds of product kernels
        x = torch.randn((tokens, 128), device=dev).to(BF16)
        ids, w = ids_of(dev, tokens, 2, 8), torch.rand((tokens, 2), device=dev)
        served(x, ids, w)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = served(x, ids, w)
        for seed in range(3):
            x.copy_(torch.randn(x.shape, device=dev))
            ids.copy_(ids_of(dev, tokens, 2, 8, seed=seed + 20))
            want = served(x, ids, w)
            y.fill_(1.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_captured_gradients(dev):
    """Forward and backward in one graph, against eager calls on the same values."""
    plan = pca.expert_sort(ids_of(dev, 60, 2, 4), 4)
    x = torch.randn((60, 96), device=dev, requires_grad=True)
    w = torch.rand((60, 2), device=dev, requires_grad=True)

    def step():
        return torch.autograd.grad(pca.expert_combine(pca.expert_dispatch(x, plan), plan, w).square().sum(), (x, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device=dev))
        want = step()
        for t in got:
            t.fill_(0.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
