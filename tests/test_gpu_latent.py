"""Latent cache, absorbed decode and expanded prefill against plain attention in
64 bits.

Tolerances of the attention outputs. With u the unit roundoff of the 16-bit
type (2^-8 for bfloat16, 2^-11 for float16) and A = sum_j softmax_j |v_j|:
rounding the weights costs u A, rounding the output u |o|. A score is an fp32
sum of D products: it is off by at most e = (D + 8) 2^-24 scale sum |q k| (in
absolute terms, natural units), which changes every weight by a factor within
1 +- 2e and the log-sum by e; 4 e A covers weights and their sum, and fp32's
other steps are within 1e-5 A. float16 weights below 2^-14 of the maximum lose
up to 2^-25 each in absolute terms: 2^-25 sum_j |v_j| more."""
from __future__ import annotations

import math

import pytest
import torch

import practice_cuda_amd as pca

pytestmark = pytest.mark.gpu

BF16, FP16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
ROUND = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}  # torch.finfo(dtype).eps / 2


def attend(q, k, v, limits, scale, dtype):
    """(out, lse, bound of out, bound of lse) of rows q over keys k; row i sees the first limits[i]."""
    q, k, v = q.double(), k.double().contiguous(), v.double().contiguous()
    seen = torch.arange(k.shape[0], device=q.device) < limits[:, None]
    scores = (q @ k.t().contiguous() * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(scores, 1)
    p = torch.exp(scores - torch.where(lse.isinf(), 0.0, lse)[:, None])
    out, size = p @ v, p @ v.abs()
    reach = (q.abs() @ k.abs().t().contiguous()).masked_fill(~seen, 0)
    e = (q.shape[1] + 8) * 2.0 ** -24 * scale * torch.nn.functional.pad(reach, (0, 1)).amax(1)
    u = ROUND[dtype]
    bound = u * size + u * out.abs() + (4 * e[:, None] + 1e-5) * size + 1e-30
    if dtype == FP16:
        bound += 2.0 ** -25 * (seen.double() @ v.abs()) + 2.0 ** -25
    return out, lse, bound, 2 * e + 1e-5 * (1 + torch.where(lse.isinf(), 0.0, lse).abs())


def near(got, want, bound, what):
    got = got.double()
    same = got == want  # -inf
    off = torch.where(same, 0.0, (got - want).abs())
    assert not torch.isnan(got).any(), f"{what}: NaN"
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times its tolerance"


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
def make_cache(g, dev, pages, page, dl, dr, dtype, fp8, junk=None):
    """A cache of random tokens, and its [places, width] values in 64 bits."""
    places = pages * page
    latent = torch.randn((places, dl), generator=g, device=dev).to(dtype)
    rope = torch.randn((places, dr), generator=g, device=dev).to(dtype)
    if fp8:
        q = pca.per_block_quant(latent, block_m=1, block_n=128)
        cache = pca.LatentCache(q.tensor.view(pages, page, dl), rope.view(pages, page, dr),
                                q.dequant_scale.view(pages, page, dl // 128))
        values = q.tensor.double().unflatten(-1, (-1, 128)) * q.dequant_scale.double().unsqueeze(-1)
        return cache, values.flatten(1), rope.double()
    return pca.LatentCache(latent.view(pages, page, dl), rope.view(pages, page, dr)), latent.double(), rope.double()


def poison(cache, places, used):
    """NaN in every place that no sequence uses."""
    free = torch.ones(places, dtype=torch.bool, device=used.device)
    free[used] = False
    cache.rope.view(places, -1)[free] = math.nan
    if cache.scale is None:
        cache.latent.view(places, -1)[free] = math.nan
    else:
        cache.latent.view(torch.uint8).view(places, -1)[free] = 0x7F
        cache.scale.view(places, -1)[free] = math.nan


def decode_case(dev, lens, new, heads, page, dtype=BF16, fp8=False, dl=512, dr=64, seed=0, strided=False, scale=0.07,
                extra_pages=3, q_std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra_pages
    cache, values, ropes = make_cache(g, dev, pages, page, dl, dr, dtype, fp8)
    order = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((len(lens), max(need) + 2), 2 ** 31 - 1, dtype=torch.int32, device=dev)  # unused: nonsense
    table[:, -1] = -5
    at, used = 0, []
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
        t = torch.arange(lens[i], device=dev)
        used.append(table[i].long()[t // page] * page + t % page)
    poison(cache, pages * page, torch.cat(used) if used else torch.empty(0, dtype=torch.long, device=dev))
    b = len(lens)
    if strided:
        ql = q_std * torch.randn((heads, b * new, dl), generator=g, device=dev)
        ql = ql.to(dtype).unflatten(1, (b, new)).permute(1, 2, 0, 3)
        qr = torch.randn((b, new, heads, dr + 24), generator=g, device=dev).to(dtype)[..., 8:8 + dr]
    else:
        ql = (q_std * torch.randn((b, new, heads, dl), generator=g, device=dev)).to(dtype)
        qr = torch.randn((b, new, heads, dr), generator=g, device=dev).to(dtype)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    kw = {}
    if strided:
        kw["out"] = torch.full((heads, b, new, dl), 7.0, dtype=dtype, device=dev).permute(1, 2, 0, 3)
    out, lse = pca.latent_decode(ql, qr, cache, table, seq, softmax_scale=scale, return_lse=True, **kw)
    assert out.shape == (b, new, heads, dl) and lse.shape == (b, new, heads)
    for i, n in enumerate(lens):
        k = torch.cat([values[used[i]], ropes[used[i]]], 1)
        q = torch.cat([ql[i], qr[i]], -1).flatten(0, 1)
        limits = (n - new + 1 + torch.arange(new, device=dev)).repeat_interleave(heads)
        want, want_lse, bound, bound_lse = attend(q, k, values[used[i]], limits, scale, dtype)
        near(out[i].flatten(0, 1), want, bound, f"out of sequence {i} ({n} tokens)")
        near(lse[i].flatten(), want_lse, bound_lse, f"lse of sequence {i} ({n} tokens)")
    again, lse2 = pca.latent_decode(ql, qr, cache, table, seq, softmax_scale=scale, return_lse=True)
    assert torch.equal(again, out) and torch.equal(lse2, lse)
    only = pca.latent_decode(ql, qr, cache, table, seq, softmax_scale=scale)
    assert torch.equal(only, out)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [1, 5, 16, 17, 32, 33, 64, 65, 100, 128, 130])
def test_decode_heads(dev, heads, fp8):
    decode_case(dev, [700, 1, 0, 33, 129], 1, heads, 64, fp8=fp8, seed=heads)


@pytest.mark.parametrize("dl,dr", [(512, 64), (256, 32)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [16, 20, 40, 128])
def test_decode_types(dev, dtype, fp8, dl, dr, heads):
    decode_case(dev, [257, 64, 1000], 1, heads, 32, dtype=dtype, fp8=fp8, dl=dl, dr=dr, seed=5)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,heads", [(2, 8), (3, 128), (4, 16), (5, 20), (7, 3)])
def test_decode_new_tokens(dev, new, heads, fp8):
    # lengths below the number of new tokens leave rows that see nothing
    decode_case(dev, [0, 1, new - 1, new, new + 1, 31, 32, 33, 500], new, heads, 16, fp8=fp8, seed=new)


@pytest.mark.parametrize("page", [1, 3, 16, 48, 64, 1000])
@pytest.mark.parametrize("heads", [16, 128])
def test_decode_pages(dev, page, heads):
    decode_case(dev, [1, 63, 64, 65, 127, 128, 333], 1, heads, page, seed=page, strided=True)
    decode_case(dev, [1, 63, 64, 65, 127, 128, 333], 1, heads, page, seed=page, strided=True, fp8=True)


@pytest.mark.parametrize("heads", [16, 30, 64, 128])
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_long(dev, heads, fp8):
    decode_case(dev, [20011], 1, heads, 64, seed=1, fp8=fp8)
    decode_case(dev, [9000, 5, 12001], 2, heads, 64, seed=2, fp8=fp8)


@pytest.mark.parametrize("heads", [8, 128])
def test_decode_many_sequences(dev, heads):
    lens = [(7 * i) % 90 for i in range(600)]
    decode_case(dev, lens, 1, heads, 16, seed=3)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype,dl,dr,page", [(BF16, 512, 64, 16), (FP16, 512, 64, 1), (BF16, 256, 32, 1),
                                              (FP16, 256, 32, 48)])
def test_decode_many_sequences_of_many_rows(dev, dtype, dl, dr, page, fp8):
    # many tiles of 128 rows: one workgroup takes a tile; page 1: more pages than are kept at hand
    lens = [0, 1] + [97 * i % 300 for i in range(195)] + [601, 333, 64]
    decode_case(dev, lens, 1, 128, page, dtype, fp8, dl, dr, seed=dl + page, q_std=4.0 if page == 1 else 1.0)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("batch,new,heads", [(3, 1, 65), (3, 2, 65), (128, 1, 66), (129, 1, 66), (97, 2, 100), (1, 3, 200)])
def test_decode_rows_of_two_workgroups(dev, batch, new, heads, fp8):
    # the last tile's second workgroup has one row, a few rows, none
    decode_case(dev, [(53 * i + 70) % 260 for i in range(batch)], new, heads, 32, fp8=fp8, seed=batch)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_decode_sharp_and_rising_scores(dev, dtype, fp8):
    # scores of +-100 and more: the running maximum moves all the time
    decode_case(dev, [3000, 40], 1, 16, 64, dtype=dtype, fp8=fp8, q_std=8.0, scale=0.5, seed=9)
    decode_case(dev, [3000, 40], 1, 128, 64, dtype=dtype, fp8=fp8, q_std=8.0, scale=0.5, seed=9)


def test_decode_minus_infinity_and_nan(dev):
    """A token that is -inf to every head takes no part; a NaN stays in its sequence."""
    g = torch.Generator(device=dev).manual_seed(0)
    cache = pca.LatentCache.empty(8, 32, device=dev)
    cache.latent.copy_(torch.randn(cache.latent.shape, generator=g, device=dev))
    cache.rope.copy_(torch.randn(cache.rope.shape, generator=g, device=dev))
    table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
    lens = torch.tensor([100, 100], dtype=torch.int32, device=dev)
    ql = torch.randn((2, 1, 16, 512), generator=g, device=dev).bfloat16()
    qr = torch.ones((2, 1, 16, 64), device=dev).bfloat16()
    want = pca.latent_decode(ql, qr, cache, table, lens, softmax_scale=0.05)
    cache.rope[5, 3] = -math.inf  # the second sequence's token 35
    got, lse = pca.latent_decode(ql, qr, cache, table, lens, softmax_scale=0.05, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.isfinite(got).all() and torch.isfinite(lse).all()
    cache.latent[5, 3] = math.nan
    got = pca.latent_decode(ql, qr, cache, table, lens, softmax_scale=0.05)
    assert torch.equal(got[0], want[0]) and torch.isnan(got[1]).all()


def test_decode_lengths_and_pages_out_of_range(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    cache = pca.LatentCache.empty(6, 16, device=dev)
    cache.latent.copy_(torch.randn(cache.latent.shape, generator=g, device=dev))
    cache.rope.copy_(torch.randn(cache.rope.shape, generator=g, device=dev))
    table = torch.tensor([[0, 1, 2], [3, 99, -1], [3, 5, 5]], dtype=torch.int32, device=dev)
    ql = torch.randn((3, 1, 16, 512), generator=g, device=dev).bfloat16()
    ql[2] = ql[1]
    qr = torch.randn((3, 1, 16, 64), generator=g, device=dev).bfloat16()
    qr[2] = qr[1]
    long = torch.tensor([2 ** 31 - 1, 48, 48], dtype=torch.int32, device=dev)
    full = torch.tensor([48, 48, 48], dtype=torch.int32, device=dev)
    a = pca.latent_decode(ql, qr, cache, table, long, softmax_scale=0.05)
    b = pca.latent_decode(ql, qr, cache, table, full, softmax_scale=0.05)
    assert torch.equal(a, b) and torch.equal(b[1], b[2])
    none = pca.latent_decode(ql, qr, cache, table, -full, softmax_scale=0.05)
    assert (none == 0).all()


def test_decode_nothing(dev):
    cache = pca.LatentCache.empty(0, 16, device=dev)
    ql, qr = torch.ones((2, 1, 16, 512), device=dev).bfloat16(), torch.ones((2, 1, 16, 64), device=dev).bfloat16()
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    for width in (0, 3):
        table = torch.zeros((2, width), dtype=torch.int32, device=dev)
        out, lse = pca.latent_decode(ql, qr, cache, table, lens, softmax_scale=1.0, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    out = pca.latent_decode(ql[:0], qr[:0], cache, table[:0], lens[:0], softmax_scale=1.0)
    assert out.shape == (0, 1, 16, 512)
    out = pca.latent_decode(ql[:, :0], qr[:, :0], cache, table, lens, softmax_scale=1.0)
    assert out.shape == (2, 0, 16, 512)


def test_decode_cache_views_of_one_buffer(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    both = torch.randn((9, 32, 576), generator=g, device=dev).bfloat16()
    split = pca.LatentCache(both[..., :512], both[..., 512:])
    apart = pca.LatentCache(both[..., :512].contiguous(), both[..., 512:].contiguous())
    table = torch.arange(9, dtype=torch.int32, device=dev).view(3, 3)
    lens = torch.tensor([96, 50, 1], dtype=torch.int32, device=dev)
    ql = torch.randn((3, 1, 128, 512), generator=g, device=dev).bfloat16()
    qr = torch.randn((3, 1, 128, 64), generator=g, device=dev).bfloat16()
    a = pca.latent_decode(ql, qr, split, table, lens, softmax_scale=0.05)
    b = pca.latent_decode(ql, qr, apart, table, lens, softmax_scale=0.05)
    assert torch.equal(a, b)


def test_decode_offsets_past_32_bits(dev):
    """Pages whose byte and element offsets pass 2^31 and 2^32."""
    pages, page = 70000, 64  # 4.6 GB of latents, 2.3 G elements
    cache = pca.LatentCache.empty(pages, page, device=dev)
    g = torch.Generator(device=dev).manual_seed(0)
    last = [pages - 1, pages // 2, 3, pages - 2]
    for p in last:
        cache.latent[p] = torch.randn((page, 512), generator=g, device=dev)
        cache.rope[p] = torch.randn((page, 64), generator=g, device=dev)
    table = torch.tensor([last], dtype=torch.int32, device=dev)
    small = pca.LatentCache(cache.latent[last].contiguous(), cache.rope[last].contiguous())
    lens = torch.tensor([250], dtype=torch.int32, device=dev)
    for heads in (16, 128):
        ql = torch.randn((1, 1, heads, 512), generator=g, device=dev).bfloat16()
        qr = torch.randn((1, 1, heads, 64), generator=g, device=dev).bfloat16()
        a = pca.latent_decode(ql, qr, cache, table, lens, softmax_scale=0.05)
        b = pca.latent_decode(ql, qr, small, torch.arange(4, dtype=torch.int32, device=dev)[None], lens,
                              softmax_scale=0.05)
        assert torch.equal(a, b)
    slots = torch.tensor([pages * page - 1, 5], device=dev)
    new = torch.randn((2, 576), generator=g, device=dev).bfloat16()
    pca.latent_append(cache, new[:, :512], new[:, 512:], slots)
    assert torch.equal(cache.latent[-1, -1], new[0, :512]) and torch.equal(cache.rope[0, 5], new[1, 512:])


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 3, 64, 1001])
@pytest.mark.parametrize("dl,dr", [(512, 64), (256, 32), (128, 8)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("fp8", [False, True])
def test_append(dev, tokens, dl, dr, dtype, fp8):
    g = torch.Generator(device=dev).manual_seed(tokens)
    page = 20
    pages = -(-tokens // page) + 2
    cache = pca.LatentCache.empty(pages, page, latent_dim=dl, rope_dim=dr, dtype=dtype, fp8=fp8, device=dev)
    for t in (cache.latent, cache.rope):
        t.view(torch.uint8).fill_(1)
    if fp8:
        cache.scale.fill_(-1.0)
    places = pages * page
    slots = torch.randperm(places, generator=g, device=dev)[:tokens]
    if tokens > 2:
        slots[1], slots[2] = -1, places + 5
    both = torch.randn((tokens, dl + dr + 1), generator=g, device=dev).to(dtype)  # rows of odd alignment
    latent, rope = both[:, :dl], both[:, dl:dl + dr]
    weight = 1 + 0.1 * torch.randn(dl, generator=g, device=dev)
    back = pca.latent_append(cache, latent, rope, slots.int() if tokens == 3 else slots, weight=weight, norm_eps=1e-5)
    assert back is cache
    kept = (slots >= 0) & (slots < places)
    at = slots[kept]
    x = latent[kept].double()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * weight.double()
    assert torch.equal(cache.rope.view(places, dr)[at], rope[kept])
    got = cache.latent.view(places, dl)[at].double() if not fp8 else \
        cache.latent.view(torch.uint8).view(places, dl)[at].view(F8).double()
    if fp8:
        scale = cache.scale.view(places, -1)[at].double()
        want = y.unflatten(-1, (-1, 128)).abs().amax(-1) / 448
        torch.testing.assert_close(scale, want, rtol=1e-5, atol=0)
        spread = want.repeat_interleave(128, -1)
        bound = (y.abs() * 2.0 ** -4).maximum(spread * 2.0 ** -10) * (1 + 1e-4) + 1e-5 * y.abs()
        assert ((got * scale.repeat_interleave(128, -1) - y).abs() <= bound).all()
    else:
        u = ROUND[dtype]
        assert ((got - y).abs() <= (u + 1e-5) * y.abs() + 2.0 ** -25).all()
    free = torch.ones(places, dtype=torch.bool, device=dev)
    free[at] = False
    assert (cache.latent.view(torch.uint8).view(places, -1)[free] == 1).all()
    assert (cache.rope.view(torch.uint8).view(places, -1)[free] == 1).all()
    if fp8:
        assert (cache.scale.view(places, -1)[free] == -1).all()


def test_append_without_norm_is_the_quantizer(dev):
    x = torch.randn((70, 512), device=dev).bfloat16()
    x[3] = 0
    rope = torch.randn((70, 64), device=dev).bfloat16()
    cache = pca.LatentCache.empty(2, 40, fp8=True, device=dev)
    pca.latent_append(cache, x, rope, torch.arange(70, device=dev))
    q = pca.per_block_quant(x, block_m=1, block_n=128)
    assert torch.equal(cache.latent.view(torch.uint8).view(80, 512)[:70], q.tensor.view(torch.uint8))
    assert torch.equal(cache.scale.view(80, 4)[:70], q.dequant_scale)
    plain = pca.LatentCache.empty(2, 40, device=dev)
    pca.latent_append(plain, x, rope, torch.arange(70, device=dev))
    assert torch.equal(plain.latent.view(80, 512)[:70], x)


# ---------------------------------------------------------------------------
# prefill
# ---------------------------------------------------------------------------
def prefill_case(dev, pairs, heads, dtype=BF16, widths=(128, 64, 128), causal=True, seed=0, spare=0, scale=None,
                 strided=False, q_std=1.0):
    dn, dr, dv = widths
    g = torch.Generator(device=dev).manual_seed(seed)
    tq, tk = sum(a for a, _ in pairs), sum(b for _, b in pairs)
    q = (q_std * torch.randn((tq + spare, heads, dn + dr), generator=g, device=dev)).to(dtype)
    kv = torch.randn((tk, heads, dn + dv), generator=g, device=dev).to(dtype)
    kr = torch.randn((tk, dr), generator=g, device=dev).to(dtype)
    kw = {}
    if strided:
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
        kr = torch.cat([kr, kr], 1)[:, :dr]
        kw["out"] = torch.full((heads, tq + spare, dv), 7.0, dtype=dtype, device=dev).transpose(0, 1)
    cu = [[0], [0]]
    for a, b in pairs:
        cu[0].append(cu[0][-1] + a)
        cu[1].append(cu[1][-1] + b)
    cu_q, cu_k = (torch.tensor(c, dtype=torch.int32, device=dev) for c in cu)
    k, v = kv[..., :dn], kv[..., dn:]
    out, lse = pca.latent_prefill(q, k, kr, v, cu_q, cu_k, softmax_scale=scale, causal=causal, return_lse=True, **kw)
    s = scale if scale is not None else (dn + dr) ** -0.5
    for i, (a, b) in enumerate(pairs):
        q0, k0 = cu[0][i], cu[1][i]
        limits = torch.arange(a, device=dev) + (b - a + 1) if causal else torch.full((a,), b, device=dev)
        for h in range(heads):
            key = torch.cat([k[k0:k0 + b, h], kr[k0:k0 + b]], 1)
            want, want_lse, bound, bound_lse = attend(q[q0:q0 + a, h], key, v[k0:k0 + b, h], limits, s, dtype)
            near(out[q0:q0 + a, h], want, bound, f"out of sequence {i} ({a}, {b}), head {h}")
            near(lse[q0:q0 + a, h], want_lse, bound_lse, f"lse of sequence {i} ({a}, {b}), head {h}")
    assert (out[tq:] == 0).all() and (lse[tq:] == -math.inf).all()
    again, lse2 = pca.latent_prefill(q, k, kr, v, cu_q, cu_k, softmax_scale=scale, causal=causal, return_lse=True)
    assert torch.equal(again, out) and torch.equal(lse2, lse)
    return out


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700])
def test_prefill_lengths(dev, n, causal):
    prefill_case(dev, [(n, n)], 3, causal=causal, seed=n)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("widths", [(128, 64, 128), (64, 32, 64)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prefill_packed(dev, dtype, widths, causal):
    # chunks after earlier keys, single queries, empty sequences, fewer keys than queries, no keys
    pairs = [(100, 100), (1, 300), (0, 50), (130, 400), (77, 20), (5, 0), (0, 0), (64, 65), (300, 300)]
    prefill_case(dev, pairs, 4, dtype=dtype, widths=widths, causal=causal, seed=1, spare=70, strided=True)


def test_prefill_many_sequences(dev):
    prefill_case(dev, [((5 * i) % 9, (5 * i) % 9 + i % 4) for i in range(700)], 1, seed=2)


@pytest.mark.parametrize("heads", [1, 7, 16, 40])
def test_prefill_heads(dev, heads):
    prefill_case(dev, [(200, 260), (50, 50)], heads, seed=heads)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prefill_sharp_scores(dev, dtype):
    prefill_case(dev, [(600, 600)], 2, dtype=dtype, q_std=8.0, scale=0.5, seed=4)


def test_prefill_long(dev):
    prefill_case(dev, [(2500, 4100)], 2, seed=5)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("widths", [(128, 64, 128), (64, 32, 64)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prefill_many_rows(dev, dtype, widths, causal):
    # ends of up to 128 rows and of more, keys before and missing, in tiles of 128 rows (256: from 8192 rows a sequence)
    pairs = [(257, 300), (129, 400), (128, 128), (256, 256), (1, 70), (30, 0), (0, 7), (385, 385), (20, 10)]
    prefill_case(dev, pairs, 56, dtype=dtype, widths=widths, causal=causal, seed=7, spare=3, strided=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prefill_many_rows_sharp_scores(dev, dtype):
    prefill_case(dev, [(900, 1000)], 74, dtype=dtype, q_std=8.0, scale=0.5, seed=8)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("widths", [(128, 64, 128), (64, 32, 64)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prefill_tiles_of_256_rows(dev, dtype, widths, causal):
    # 8192 rows a sequence and more on average, most of them behind the last sequence
    pairs = [(257, 300), (129, 400), (128, 128), (256, 256), (1, 70), (30, 0), (0, 7), (385, 385), (900, 1100)]
    prefill_case(dev, pairs, 2, dtype=dtype, widths=widths, causal=causal, seed=9, spare=9 * 8192, strided=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prefill_tiles_of_256_rows_sharp_scores(dev, dtype):
    prefill_case(dev, [(900, 1000)], 2, dtype=dtype, q_std=8.0, scale=0.5, seed=8, spare=65536)


@pytest.mark.parametrize("n", [63, 64, 65])
def test_prefill_tiles_of_256_rows_in_many_sequences(dev, n):
    prefill_case(dev, [((37 * i) % 350, (37 * i) % 350 + i % 6) for i in range(n)], 1, seed=n, spare=n * 8192)


@pytest.mark.parametrize("n", [62, 63, 64, 65])
@pytest.mark.parametrize("heads", [1, 64])
def test_prefill_sequences_of_a_wave(dev, n, heads):
    # up to 63 sequences a wave finds its tile alone
    prefill_case(dev, [((37 * i) % 35 + (0 if heads == 1 else 2), (37 * i) % 35 + i % 6) for i in range(n)], heads,
                 seed=n)


def test_scales_of_zero_and_below(dev):
    prefill_case(dev, [(100, 130), (3, 3)], 2, scale=0.0, seed=1)
    decode_case(dev, [300, 1, 0], 2, 5, 16, scale=0.0, seed=1)
    decode_case(dev, [300, 1, 0], 1, 100, 16, fp8=True, scale=0.0, seed=1)
    g = torch.Generator(device=dev).manual_seed(3)
    q, k, v, kr = (torch.randn(s, generator=g, device=dev).bfloat16()
                   for s in ((90, 3, 192), (90, 3, 128), (90, 3, 128), (90, 64)))
    cu = torch.tensor([0, 90], dtype=torch.int32, device=dev)
    a, b = (pca.latent_prefill(x, k, kr, v, cu, cu, softmax_scale=s) for x, s in ((q, -0.07), (-q, 0.07)))
    assert torch.equal(a, b)
    cache = pca.LatentCache.empty(4, 64, device=dev)
    cache.latent.normal_(generator=g)
    cache.rope.normal_(generator=g)
    table, lens = torch.arange(4, dtype=torch.int32, device=dev)[None], torch.tensor([222], dtype=torch.int32, device=dev)
    for heads in (16, 128):
        ql, qr = (torch.randn((1, 1, heads, n), generator=g, device=dev).bfloat16() for n in (512, 64))
        a = pca.latent_decode(ql, qr, cache, table, lens, softmax_scale=-0.07)
        assert torch.equal(a, pca.latent_decode(-ql, -qr, cache, table, lens, softmax_scale=0.07))


def test_rows_off_their_alignment_are_refused(dev):
    cu = torch.tensor([0, 8], dtype=torch.int32, device=dev)
    q = torch.zeros((8, 2, 196), device=dev).bfloat16()[..., 4:]
    k, kr = torch.zeros((8, 2, 128), device=dev).bfloat16(), torch.zeros((8, 64), device=dev).bfloat16()
    with pytest.raises(ValueError, match="q"):
        pca.latent_prefill(q, k, kr, k, cu, cu)
    q = q.contiguous()
    with pytest.raises(ValueError, match="v"):
        pca.latent_prefill(q, k, kr, torch.zeros((8, 2, 132), device=dev).bfloat16()[..., :128], cu, cu)
    cache = pca.LatentCache.empty(2, 16, device=dev)
    table, lens = torch.zeros((1, 2), dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    ql, qr = torch.zeros((1, 1, 2, 516), device=dev).bfloat16(), torch.zeros((1, 1, 2, 64), device=dev).bfloat16()
    with pytest.raises(ValueError, match="q_latent"):
        pca.latent_decode(ql[..., 4:], qr, cache, table, lens, softmax_scale=1.0)
    odd = pca.LatentCache(torch.zeros((2, 16, 516), device=dev).bfloat16()[..., :512], cache.rope)
    with pytest.raises(ValueError, match="latent"):
        pca.latent_decode(ql[..., :512].contiguous(), qr, odd, table, lens, softmax_scale=1.0)


def test_prefill_nothing(dev):
    q = torch.ones((5, 2, 192), device=dev).bfloat16()
    k = torch.ones((0, 2, 128), device=dev).bfloat16()
    kr = torch.ones((0, 64), device=dev).bfloat16()
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    out, lse = pca.latent_prefill(q, k, kr, k, zero, zero, return_lse=True)  # no sequences
    assert (out == 0).all() and (lse == -math.inf).all()
    out = pca.latent_prefill(q[:0], k, kr, k, zero, zero)
    assert out.shape == (0, 2, 128)
    # offsets beyond the tensors are cut to them
    q = torch.randn((50, 2, 192), device=dev).bfloat16()
    k, v = torch.randn((50, 2, 128), device=dev).bfloat16(), torch.randn((50, 2, 128), device=dev).bfloat16()
    kr = torch.randn((50, 64), device=dev).bfloat16()
    good = torch.tensor([0, 50], dtype=torch.int32, device=dev)
    far = torch.tensor([-3, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    assert torch.equal(pca.latent_prefill(q, k, kr, v, good, good), pca.latent_prefill(q, k, kr, v, far, far))


def test_prefill_nan_stays_in_its_sequence(dev):
    q, k, v = (torch.randn((128, 2, w), device=dev).bfloat16() for w in (192, 128, 128))
    kr = torch.randn((128, 64), device=dev).bfloat16()
    cu = torch.tensor([0, 40, 128], dtype=torch.int32, device=dev)
    want = pca.latent_prefill(q, k, kr, v, cu, cu)
    v[40:], k[40:] = math.nan, math.nan
    got = pca.latent_prefill(q, k, kr, v, cu, cu)
    assert torch.equal(got[:40], want[:40]) and torch.isnan(got[40:]).all()


# ---------------------------------------------------------------------------
# both forms, streams, graphs
# ---------------------------------------------------------------------------
def test_absorbed_equals_expanded(dev):
    """One new token over the cache gives what the last row of the prompt gives."""
    g = torch.Generator(device=dev).manual_seed(0)
    n, heads = 150, 4
    c = torch.randn((n, 512), generator=g, device=dev).bfloat16()
    kr = torch.randn((n, 64), generator=g, device=dev).bfloat16()
    wk, wv = (torch.randn((heads, 128, 512), generator=g, device=dev) / 512 ** 0.5 for _ in range(2))
    q = torch.randn((n, heads, 192), generator=g, device=dev).bfloat16()
    k = torch.stack([(c.float() @ w.t().contiguous()).bfloat16() for w in wk], 1)
    v = torch.stack([(c.float() @ w.t().contiguous()).bfloat16() for w in wv], 1)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    expanded = pca.latent_prefill(q, k, kr, v, cu, cu)[-1].float()
    cache = pca.LatentCache.empty(5, 32, device=dev)
    pca.latent_append(cache, c, kr, torch.arange(n, device=dev))
    ql = torch.stack([q[-1, h, :128].float() @ wk[h] for h in range(heads)]).bfloat16()
    table = torch.arange(5, dtype=torch.int32, device=dev)[None]
    o = pca.latent_decode(ql[None, None], q[None, -1:, :, 128:], cache, table,
                          torch.tensor([n], dtype=torch.int32, device=dev), softmax_scale=192 ** -0.5)
    absorbed = torch.stack([o[0, 0, h].float() @ wv[h].t().contiguous() for h in range(heads)])
    # the two forms round different intermediates to bfloat16
    assert (absorbed - expanded).abs().max() <= 0.05 * expanded.abs().max()


def test_streams_and_graph(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    cache = pca.LatentCache.empty(40, 64, fp8=True, device=dev)
    tokens = torch.randn((2500, 576), generator=g, device=dev).bfloat16()
    pca.latent_append(cache, tokens[:, :512], tokens[:, 512:], torch.arange(2500, device=dev))
    table = torch.arange(40, dtype=torch.int32, device=dev).view(2, 20)
    lens = torch.tensor([1200, 900], dtype=torch.int32, device=dev)
    ql = torch.randn((2, 1, 128, 512), generator=g, device=dev).bfloat16()
    qr = torch.randn((2, 1, 128, 64), generator=g, device=dev).bfloat16()
    slot = torch.tensor([1199, 20 * 64 + 899], device=dev)
    new = torch.randn((2, 576), generator=g, device=dev).bfloat16()

    def step():
        pca.latent_append(cache, new[:, :512], new[:, 512:], slot)
        return pca.latent_decode(ql, qr, cache, table, lens, softmax_scale=0.07, return_lse=True)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):  # other tokens and lengths between replays
        new.copy_(torch.randn_like(new))
        lens.copy_(torch.tensor([1200 - 300 * k, 5 + 200 * k], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
