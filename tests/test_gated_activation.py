"""The activations of the gated product: GELU's polynomial as the source holds it, in f32, and both functions over their tails."""
import math
import os
import re

import pytest
import torch

from scratchtape_amd import build, quant8
from quant8_oracle import U


def test_gelu_polynomial():
    """erfc(z) exp(z^2) = t P(t), t = 1 / (1 + z / 2), within 4.6e-8 with the source's numbers as f32 holds them, for z up to 14."""
    body = open(os.path.join(build.CSRC, "matmul8.hip")).read().split("__device__ __forceinline__ float gated(")[1].split("\n}\n")[0]
    f32 = lambda text: float(torch.tensor(float(text), dtype=torch.float32))
    slope = f32(re.search(r"rcpf\(__builtin_fmaf\(([\d.]+)f, __builtin_fabsf\(g\), 1\.f\)\)", body).group(1))
    numbers = [f32(v) for v in re.findall(r"float p = (-?[\d.]+)f;|fmaf\(p, t, (-?[\d.]+)f\)", body) for v in v if v]
    assert len(numbers) == 9
    g = torch.linspace(0, 14 * math.sqrt(2), 400001, dtype=torch.float64)
    t = 1 / (1 + slope * g)
    p = torch.zeros_like(t)
    for v in numbers:
        p = p * t + v
    assert float((t * p / torch.special.erfcx(g / math.sqrt(2)) - 1).abs().max()) < 4.6e-8


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_tails(dev, activation):
    """act(g) for u = 1 over g of all sizes, relative errors: those of the f32 operations one after the other.  The argument of exp2 is off by its
    product's roundings and its constant's, 1.22 U (silu) and 2.22 U (gelu) of itself, exp2 and the reciprocal by 2 U, the polynomial
    by 0.8 U, the rounding of t (2 U and 1 U before it) and its steps by 8 U; what exp2 gives below 2^-126 may be 0."""
    most = 14.0 if activation == "gelu" else 80.0
    size = torch.logspace(-8, math.log10(most / 127), 150)
    x = torch.zeros(127, 16, dtype=torch.int8)
    x[:, 0], x[:, 1] = torch.arange(1, 128), 1
    w = torch.zeros(600, 16, dtype=torch.int8)
    w[:150, 0], w[150:300, 0], w[300:, 1] = 1, -1, 1
    ws = torch.cat((size, size, torch.ones(300)))
    got = quant8.gated_8bit(x.to(dev), torch.ones(127, device=dev), w.to(dev), ws.to(dev), activation=activation, dtype=torch.float32).cpu().double()
    g = (torch.arange(1.0, 128)[:, None] * torch.cat((size, -size))).double()  # (the product in f32)
    z = g.abs()
    if activation == "silu":
        want = g * torch.sigmoid(g)
        rel = (1.22 * z * torch.sigmoid(-g) + 7) * U
    else:
        tail = 0.5 * torch.special.erfc(z / math.sqrt(2))
        want = g * torch.where(g < 0, tail, 1 - tail)
        rel = torch.where(g < 0, torch.ones_like(g), tail / (1 - tail)) * (1.11 * z * z + 16) * U + 2 * U
    assert bool(((got - want).abs() <= 1.01 * rel * want.abs() + 2.0 ** -125 * z).all()), float(((got - want).abs() / (rel * want.abs())).nan_to_num().max())
