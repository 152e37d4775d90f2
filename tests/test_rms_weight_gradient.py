"""The norm's weight gradient over many rows: its error is that of sums in 64 bits, however many rows a lane adds up.

dw = sum over rows of t = dy xh.  In f32 are rounded: xh, each workgroup's part and dw itself.  A rounding is off by at most U of its
value, and with values of all mantissas by U / sqrt 3 of it at most in the root of the mean square; the errors are independent and the
terms' signs random, so that the parts' squares add up to those of the terms, as dw's do: off by U / sqrt 3 sqrt(t^2 + parts^2 + dw^2)
= U of dw in the root of the mean square, over columns.  The bound is 1.25 U.  A chain of L additions in f32 adds U sqrt(L / 6) to that in
the same measure (U / sqrt 3 of partial sums that grow from nothing to a part), 0.6 to 0.75 of it for mantissas spread evenly."""
import pytest
import torch

from scratchtape_amd import rows
from quant8_oracle import U

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BOUND = 1.25 * U


def off(got, want):
    """The error of dw, relative, in the root of the mean square."""
    return float((got.double() - want).norm() / want.norm())


def inputs(n, d, t, dev):
    g = torch.Generator(dev).manual_seed(n + d)
    dy, h = (torch.randn(n, d, generator=g, device=dev, dtype=torch.float32).to(t) for _ in range(2))
    return dy, h, torch.rand(n, generator=g, device=dev) + 0.5


def exact(dy, h, rstd):
    want = torch.zeros(dy.shape[1], dtype=torch.float64, device=dy.device)
    for i in range(0, len(dy), 4096):
        part = slice(i, i + 4096)
        want += (dy[part].double() * h[part].double() * rstd[part].double()[:, None]).sum(0)
    return want


@pytest.mark.parametrize("t", sorted(TYPES))
def test_the_bound_tells_chains_apart(t):
    """Parts of 64 rows, a row lane each: summed in 64 bits within the bound, in f32 (a mistake planted here) beyond it."""
    dy, h, rstd = inputs(64 * 128, 512, TYPES[t], "cpu")
    want = exact(dy, h, rstd)
    products = (dy.double() * (h.float() * rstd[:, None]).double()).view(64, 128, 512)
    assert off(products.sum(0).float().double().sum(0).float(), want) < BOUND
    chain = torch.zeros(128, 512)
    for row in products:
        chain = (chain.double() + row).float()
    assert off(chain.double().sum(0).float(), want) > 1.5 * BOUND


# Every kernel of the backward, 64 rows and more a row lane (for the widest 400 a part)
@pytest.mark.gpu
@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,d", [(131072, 256), (131072, 511), (131072, 1000), (131072, 2000), (65536, 3000), (32768, 4096), (16384, 8000), (16384, 16000),
                                 (25600, 17000)])
def test_weight_gradient_of_many_rows(dev, n, d, t):
    dy, h, rstd = inputs(n, d, TYPES[t], dev)
    want = exact(dy, h, rstd)
    weights = torch.ones(d, device=dev)
    for w in {weights.dtype: weights, TYPES[t]: weights.to(TYPES[t])}.values():
        dx, dw = rows.rms_norm_backward(dy, h, rstd, w)
        assert off(dw, want) < BOUND
        del dx
