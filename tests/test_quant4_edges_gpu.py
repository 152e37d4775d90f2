"""Products with 4-bit weights where the definition's sums are infinite, or finite although sums that the kernel takes on the way
are not: what sum over l of x[l] w[l] is, in 64 bits rounded to the type."""
import math

import pytest
import torch

import quant4_oracle as oracle
from scratchtape_amd import quant4
from test_quant4_gpu import TYPES, check_product

pytestmark = pytest.mark.gpu
SHAPES = [(1, 256, 50, 32), (3, 96, 17, 32), (16, 1024, 200, 128), (20, 640, 100, 64), (5, 192, 8300, 64), (1, 8192, 70, 128), (33, 128, 40, 32)]


def made(n, k, group, shift, dev):
    g = torch.Generator().manual_seed(n + k)
    return quant4.quantize_4bit((torch.randn(n, k, generator=g) * 0.05 + shift).to(dev), group)


def values_of(codes, scales):
    n, groups = scales.shape[:2]
    return (oracle.unpack(codes.cpu()).view(n, groups, -1) * scales[..., :1].cpu().double() + scales[..., 1:].cpu().double()).view(n, -1)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("m,k,n,group", SHAPES)
def test_infinite_rows(dev, m, k, n, group, t):
    """A row with one infinity is infinite by the weight's sign, one with several by their agreement, one with a NaN is NaN; the
    others are as without them.  With ReLU minus infinity is 0."""
    codes, scales = made(n, k, group, 0.0, dev)
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, k, generator=g).to(TYPES[t])
    rows = [0, m // 2, m - 1]
    x[rows[0], k - 1] = math.inf
    if m > 2:
        x[rows[1], 0], x[rows[1], k // 2] = -math.inf, math.inf
        x[rows[2], 5], x[rows[2], 6] = -math.inf, math.nan
    w = values_of(codes, scales)
    want = (x.double()[:, None] * w[None]).sum(-1) if m * k * n < 1 << 23 else torch.stack([(r.double() * w).sum(-1) for r in x])
    bias = torch.randn(n, generator=g).to(dev)
    got = quant4.matvec_4bit(x.to(dev), codes, scales, bias=bias)
    bad = ~torch.isfinite(want)
    assert torch.equal(got.cpu().double()[bad].nan_to_num(7.0), want[bad].nan_to_num(7.0))
    assert bool(bad[rows].all()) and (m == 1 or bool(want[rows[0]].isinf().all()))
    clean = [r for r in range(m) if r not in rows]
    if clean:
        check_product(x[clean].to(dev), codes, scales, bias, False, got[clean])
    got = quant4.matvec_4bit(x.to(dev), codes, scales, bias=bias, relu=True).cpu().double()
    assert torch.equal(got[bad].nan_to_num(7.0), want[bad].clamp(min=0).nan_to_num(7.0))


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n,group", SHAPES)
def test_large_rows_of_small_weights(dev, m, k, n, group, t):
    """Rows near the type's largest value: products with weights below 1/8 are finite, sums of 16 + c times them are not."""
    for shift in (0.0, 0.06):
        codes, scales = made(n, k, group, shift, dev)
        g = torch.Generator().manual_seed(m)
        x = (torch.randn(m, k, generator=g).clamp(-3, 3) * (2.0 ** 125 / k ** 0.5)).to(TYPES[t])
        x[0] = x[0].sign() * 3e38 / (30 if k < 300 else 300)
        check_product(x.to(dev), codes, scales, None, False, quant4.matvec_4bit(x.to(dev), codes, scales))


def test_a_weight_of_zero_and_an_infinite_row(dev):
    """0 times an infinity is no number, and the groups beside it do not matter."""
    w = torch.linspace(-1, 1, 64).repeat(3, 2)
    w[1, 64:] = 0.0
    codes, scales = quant4.quantize_4bit(w.to(dev), 64)
    x = torch.ones(1, 128)
    x[0, 100] = math.inf
    for t in TYPES.values():
        y = quant4.matvec_4bit(x.to(t).to(dev), codes, scales).cpu()
        assert bool(y[0, 1].isnan()) and bool((y[0, [0, 2]] == math.inf).all())


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n", [(1, 4096), (1, 4097), (5, 8192), (16, 8193), (17, 2048), (17, 2049), (32, 4096), (33, 2731), (31, 4097), (70, 300),
                                 (130, 517)])
def test_products_around_the_widths_of_tiles(dev, m, n, group, t):
    """Sizes at which a workgroup takes 16, 32 and 64 rows of weights, and one and two blocks of x: the same sums, held to 64 bits,
    and for a row to the bits that it has alone."""
    codes, scales = made(n, 384, group, 0.01, dev)
    x = torch.randn(m, 384, generator=torch.Generator().manual_seed(n)).to(TYPES[t]).to(dev)
    got = quant4.matvec_4bit(x, codes, scales)
    check_product(x, codes, scales, None, False, got)
    assert torch.equal(quant4.matvec_4bit(x[m // 2:m // 2 + 1], codes, scales)[0], got[m // 2])
