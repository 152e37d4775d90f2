"""How many bits of f32 and f16 rows the 4-bit products and the cache attention keep: the root of the mean squared error, which a lost
part of a row or of a weight raises far above what rounding leaves (the worst-case bounds of the other tests would hide it).

The CPU tests plant the loss in the oracle: the same sums in 64 bits with rows and weights held in as many parts as the kernels
take pass the bounds, with a part fewer they do not.

f32 attention: queries and weights in two f16 parts (22 bits), scores and sums in f32.  A score of size up to 16 (log2) is off by
2^-21 a rounding at the most; eight of them are allowed.  f16 and bf16 outputs of few rows: the error of the output's own rounding is
most of it; 1.15 times that is allowed (one f16 part of the weights: 1.4 for f16).  f32 products: three bf16 parts (24 bits) and f32
sums; 2^-20 of the outputs' size is allowed, 16 roundings."""
import math

import pytest
import torch

import quant4_oracle as oracle

ATTENTION, ROUNDING, PRODUCT = 8 * 2.0 ** -21, 1.15, 2.0 ** -20
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(1, 32, 1), (4, 64, 1), (1, 96, 5), (3, 128, 1), (2, 192, 2), (1, 256, 40), (2, 64, 150), (4, 128, 130)]  # share, hd, new


def rms(x):
    return float(x.double().square().mean().sqrt())


def made(share, hd, new, t, seed=0, length=777):
    """One sequence and key head: q [new, share, hd], and codes, scales, values of its keys and values."""
    g = torch.Generator().manual_seed(seed * 1000 + hd + new)
    q = (torch.randn(new, share, hd, generator=g) * 2).to(TYPES[t])
    kv = [oracle.quantise(torch.randn(length, hd, generator=g)) for _ in range(2)]
    return q, kv


def attend(q, kv, parts_q, parts_w):
    """softmax(q k^T / sqrt(hd)) v in 64 bits (parts 0), or with rows and weights in f16 parts as the kernel holds them."""
    new, share, hd = q.shape
    (kc, ka, kb), (vc, va, vb) = kv
    length = kc.shape[0]
    y = q.double()
    held = y
    if parts_q:
        lift = 15 - torch.floor(torch.log2(y.abs().amax(-1, keepdim=True))) - 1
        x = y * 2.0 ** lift
        high = x.half().double()
        held = (high + ((x - high).half().double() if parts_q == 2 else 0)) * 2.0 ** -lift
    z = ((held @ (kc - 8).double().t()) * ka[:, 0] + y.sum(-1, keepdim=True) * (kb + 8 * ka)[:, 0]) / math.sqrt(hd) / math.log(2)
    seen = torch.arange(length)[None] <= (length - new + torch.arange(new))[:, None]
    z = z.masked_fill(~seen[:, None], -math.inf)
    top = (z + torch.log2(va[:, 0])).amax(-1, keepdim=True).ceil() - 7
    p = 2.0 ** (z - top)
    w = p * va[:, 0]
    if parts_w:
        high = w.half().double()
        w = high + ((w - high).half().double() if parts_w == 2 else 0)
    return (w @ (vc - 8).double() + p @ (vb + 8 * va).expand(-1, hd)) / p.sum(-1, keepdim=True)


def attention_error(got, exact, t):
    """Over the bound, and below 1 where it holds."""
    if t == "f32":
        return rms(got.double() - exact) / rms(exact) / ATTENTION
    return rms(got.double() - exact) / rms(exact.to(TYPES[t]).double() - exact) / ROUNDING


@pytest.mark.parametrize("share,hd,new", SHAPES)
def test_a_lost_part_shows_in_attention(share, hd, new):
    q, kv = made(share, hd, new, "f32")
    exact = attend(q, kv, 0, 0)
    assert attention_error(attend(q, kv, 2, 2).float(), exact, "f32") < 0.25
    assert attention_error(attend(q, kv, 1, 2).float(), exact, "f32") > 4
    assert attention_error(attend(q, kv, 2, 1).float(), exact, "f32") > 4
    q, kv = made(share, hd, new, "f16")
    exact = attend(q, kv, 0, 0)
    assert attention_error(attend(q, kv, 1, 2).half(), exact, "f16") < 1
    if share * new * hd >= 480:  # (fewer outputs scatter too far for a factor of 1.2)
        assert attention_error(attend(q, kv, 1, 1).half(), exact, "f16") > 1
    q, kv = made(share, hd, new, "bf16")
    assert attention_error(attend(q, kv, 1, 1).bfloat16(), attend(q, kv, 0, 0), "bf16") < 1


PRODUCTS = [(1, 256, 1024, 64), (3, 96, 130, 32), (16, 4096, 515, 32), (1, 8192, 77, 128), (17, 640, 255, 128), (2, 1408, 4255, 128), (5, 32, 9000, 32)]


def product_case(m, k, n, group):
    g = torch.Generator().manual_seed(m + k + n)
    c, scale, lo = oracle.quantise(torch.randn(n, k // group, group, generator=g) * 0.05)
    x = torch.randn(m, k, generator=g)
    return x, c, scale, lo, (c * scale + lo).view(n, k)


def bf16_parts(x, parts):
    """x as the sum of its first `parts` parts of 8 bits, taken off without rounding."""
    rest, total = x.clone(), torch.zeros_like(x, dtype=torch.float64)
    for _ in range(parts):
        part = (rest.view(torch.int32) & -65536).view(torch.float32)
        total += part.double()
        rest = rest - part
    return total


@pytest.mark.parametrize("m,k,n,group", PRODUCTS)
def test_a_lost_part_shows_in_products(m, k, n, group):
    x, _, _, _, w = product_case(m, k, n, group)
    exact = x.double() @ w.t()
    assert torch.equal(bf16_parts(x, 3), x.double())
    assert rms(bf16_parts(x, 2) @ w.t() - exact) > 2 * PRODUCT * rms(exact)


# ---- the kernels -------------------------------------------------------------------------------------------------

def cached(kv, page, dev):
    """The keys and values in a cache of one head, its pages in reverse order, and its table."""
    from scratchtape_amd.kv4 import KvCache4bit

    length, hd = kv[0][0].shape
    per = -(-length // page)
    cache, table = KvCache4bit.empty(per, 1, page, hd, dev), torch.arange(per - 1, -1, -1, dtype=torch.int32, device=dev)[None]
    at = torch.arange(length, device=dev)
    p, slot = table[0].long()[at // page], at % page
    for (c, scale, lo), codes, scales in ((kv[0], cache.k_codes, cache.k_scales), (kv[1], cache.v_codes, cache.v_scales)):
        codes[p, 0, slot] = oracle.pack(c).to(dev)
        scales[p, 0, slot] = torch.cat((scale, lo), -1).float().to(dev)
    return cache, table


@pytest.mark.gpu
@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("length", [777, 5000])
@pytest.mark.parametrize("share,hd,new", SHAPES)
def test_attention_keeps_its_bits(dev, share, hd, new, length, t):
    q, kv = made(share, hd, new, t, length=length)
    cache, table = cached(kv, 32, dev)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    got = cache.attention(q.to(dev), table, ints(0, new), ints(length)).cpu()
    exact = attend(q, kv, 0, 0)
    # f16 rows of more than 64 rows a sequence hold their weights in one part: 1.41 times the output's rounding, and a tenth.
    allowed = 1.55 / ROUNDING if t == "f16" and share * new >= 64 and hd <= 128 else 1.0
    assert attention_error(got, exact, t) < allowed


@pytest.mark.gpu
@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("m,k,n,group", PRODUCTS)
def test_products_keep_their_bits(dev, m, k, n, group, t):
    from scratchtape_amd import quant4

    x, c, scale, lo, w = product_case(m, k, n, group)
    x = x.to(TYPES[t])
    got = quant4.matvec_4bit(x.to(dev), oracle.pack(c.view(n, k)).to(dev), torch.cat((scale, lo), -1).float().to(dev)).cpu().double()
    exact = x.double() @ w.t()
    if t == "f32":
        assert rms(got - exact) <= PRODUCT * rms(exact)
    else:
        assert rms(got - exact) <= 1.02 * rms(exact.to(TYPES[t]).double() - exact)
