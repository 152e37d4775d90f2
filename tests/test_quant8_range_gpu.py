"""8-bit products whose result is in f32's range and whose sum times the row's scale is not, on each of the kernels."""
import math

import pytest
import torch

from scratchtape_amd import quant8
import quant8_oracle as oracle
import test_quant8_tiles_gpu as tiles

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
LINEAR = [s[:4] for s in tiles.LINEAR if s[1:4] in ((2300, 4096, 11000), (700, 16, 20000), (3000, 100, 5001), (129, 4100, 4099), (100, 131072, 70),
                                                   (33, 4096, 515), (17, 4111, 30000), (7, 2050, 40), (3, 1000, 50000), (1, 65536, 300))]
GATED = [s[:4] for s in tiles.GATED if s[1:4] in ((1000, 4096, 12300), (130, 4096, 12288), (90, 333, 6001), (40, 512, 20000), (30, 500, 700),
                                                 (4, 3000, 3001), (1, 8192, 4000))]


def operands(m, k, n, dev):
    """Rows of x of all scales up to f32's largest (sums times the scale pass it), channels so small that results are in range."""
    x, xs, w, ws = tiles.operands(m, k, n, m + n, dev)
    xs = (0.5 + 25 * xs) * 2.0 ** (torch.linspace(0, 127, m, device=dev).round() if m > 1 else torch.full((1,), 127.0, device=dev))
    assert bool(xs.isfinite().all()) and float(xs.max()) >= 2.0 ** 126
    return x, xs, w, ws * 2.0 ** -118


def test_every_kernel_is_here():
    assert {s[0] for s in LINEAR} >= {"large", "middle", "small", "deep", "few", "one"}
    assert {s[0] for s in GATED} >= {"large", "middle", "low", "deep_low", "few", "one"}


@pytest.mark.parametrize("kernel,m,k,n", LINEAR)
def test_large_scales(dev, kernel, m, k, n):
    assert quant8.product_plan(m, k, n)[0] == kernel
    x, xs, w, ws = operands(m, k, n, dev)
    bias = torch.randn(n, generator=torch.Generator(dev).manual_seed(1), device=dev)
    for t, b, relu in ((F32, None, False), (F32, bias, True), (BF16, bias, False)):
        y, tol = tiles.product(x, xs, w, ws, b)
        assert float(y.abs().max()) < torch.finfo(t).max / 2
        tiles.close(quant8.matmul_8bit(x, xs, w, ws, bias=b, relu=relu, dtype=t), y.clamp(min=0) if relu else y, tol)


@pytest.mark.parametrize("kernel,m,k,n", GATED)
def test_large_scales_gated(dev, kernel, m, k, n):
    assert quant8.product_plan(m, k, n, gated=True)[0] == kernel
    x, xs, w, ws = operands(m, k, 2 * n, dev)
    y, tol = tiles.product(x, xs, w, ws, None)
    want, off = oracle.gated((y[:, :n], tol[:, :n]), (y[:, n:], tol[:, n:]), "silu")
    tiles.close(quant8.gated_8bit(x, xs, w, ws, dtype=F32), want, off)


def test_large_scales_in_slices(dev):
    m, k, n = 100, 8192, 60
    assert quant8.product_plan(m, k, n, gated=True)[1] > 1
    x, xs, w, ws = operands(m, k, 2 * n, dev)
    y, tol = tiles.product(x, xs, w, ws, None)
    want, off = oracle.gated((y[:, :n], tol[:, :n]), (y[:, n:], tol[:, n:]), "gelu")
    tiles.close(quant8.gated_8bit(x, xs, w, ws, activation="gelu", dtype=F32), want, off)


def test_large_scales_of_unaligned_rows(dev):
    m, k, n = 70, 200, 90
    x, xs, w, ws = operands(m, k, n, dev)
    off = torch.empty(m * (k + 1) + 1, dtype=torch.int8, device=dev)[1:].view(m, k + 1)[:, :k]
    off.copy_(x)
    y, tol = tiles.product(x, xs, w, ws, None)
    tiles.close(quant8.matmul_8bit(off, xs, w, ws, dtype=F32), y, tol)


@pytest.mark.parametrize("m", [1, 7, 40, 200])
def test_zero_sums_and_scales_that_are_not_finite(dev, m):
    """Sums of 0 between scales whose product is past f32's range are 0; NaN in either scale is NaN; a result past the range is infinite."""
    k, n = 512, 48
    x, w = (torch.zeros(rows, k, dtype=torch.int8, device=dev) for rows in (m, n))
    xs, ws = (torch.full((rows,), 2.0 ** 120, device=dev) for rows in (m, n))
    w[5], ws[7] = 3, math.nan
    got = quant8.matmul_8bit(x, xs, w, ws, dtype=F32)
    assert bool(got[:, 7].isnan().all()) and not bool(got[:, :7].any()) and not bool(got[:, 8:].any())
    x[0, 3], xs[-1] = -1, math.nan if m > 1 else xs[-1]
    got = quant8.matmul_8bit(x, xs, w, ws, dtype=F32)
    assert bool(got[0, 5] == -math.inf) and not bool(got[0, :5].any())
    assert m == 1 or bool(got[-1].isnan().all())
