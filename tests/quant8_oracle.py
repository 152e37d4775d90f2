"""The 8-bit row format, products of 8-bit rows, the gated product, and the root-mean-square norm with its gradients in 64
bits, for the tests: written from the definitions, with how far 32-bit arithmetic may take a result from them."""
import math

import torch

U = 2.0 ** -24  # half a unit of f32's last place


def half_step(t):
    """(relative, absolute) rounding to a type: half a step of normal and of subnormal numbers."""
    info = torch.finfo(t)
    return info.eps / 2, info.smallest_normal * info.eps / 2


def rounded(y, t):
    rel, tiny = half_step(t)
    return rel * y.abs() + tiny


def quantise(t):
    """Rows t [n, k] (float64) -> codes (int64), a = max |t| (NaN where a row is not finite)."""
    a = t.abs().amax(-1)
    bad = ~torch.isfinite(t).all(-1)
    codes = torch.where(((a > 0) & ~bad)[:, None], torch.round(t * 127 / a[:, None]), torch.zeros_like(t))
    return codes.nan_to_num(0).long(), torch.where(bad, torch.full_like(a, math.nan), a)


def product(x, x_scales, w, w_scales, bias=None):
    """(x w^T) xs ws + bias for int8 codes, and what f32 may be off: the sum to f32, two products by scales, the addition."""
    s = (x.cpu().double() @ w.cpu().double().t()) * x_scales.cpu().double()[:, None] * w_scales.cpu().double()
    y = s if bias is None else s + bias.cpu().double()
    return y, 2.01 * U * s.abs() + U * y.abs() + 2.0 ** -148


def gated(g, u, activation):
    """act(g) u for products with their tolerances."""
    (g, eg), (u, eu) = g, u
    act = g / (1 + torch.exp(-g)) if activation == "silu" else 0.5 * g * torch.special.erfc(-g / math.sqrt(2))
    act = torch.where(torch.isneginf(g), torch.full_like(g, math.nan), act)
    # |act'| <= 1.13; the function itself within 8 U of its value, and (the argument of erfc, the tail of exp) 2 U
    ea = 1.13 * eg + 8 * U * act.abs() + 2 * U
    return act * u, 1.01 * (ea * u.abs() + act.abs() * eu + ea * eu) + 2 * U * (act * u).abs()


def norm(x, residual, weight, eps):
    """h (in x's type), rstd, y and t = h weight, in 64 bits from h on."""
    h = x.cpu() if residual is None else (x.cpu().double() + residual.cpu().double()).to(x.dtype)
    hd = h.double()
    rstd = 1 / torch.sqrt(hd.square().mean(-1) + torch.tensor(eps, dtype=torch.float32).double())
    t = hd * weight.cpu().double()
    return h, rstd, t * rstd[:, None], t


def norm_backward(dy, h, rstd, weight, dh):
    """dx and dweight with their tolerances."""
    dy, h, w, r = dy.cpu().double(), h.cpu().double(), weight.cpu().double(), rstd.cpu().double()[:, None]
    xh, g = h * r, dy * w
    mean, size = (g * xh).mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    dx = r * (g - xh * mean)
    # g to f32, xh, the mean (its products to f32, itself), their product and difference, the product with rstd
    off = r * (3 * U * g.abs() + 5 * U * xh.abs() * size)
    if dh is not None:
        dx = dx + dh.cpu().double()
    dw, sizes = (dy * xh).sum(0), (dy * xh).abs().sum(0)
    # a thread's chain of f32 additions: its rows and the other row lanes', at most 36 and a 1024th of all
    return (dx, 1.01 * off + U * dx.abs() + 2.0 ** -140), (dw, (38 + h.shape[0] / 1024) * U * sizes + 2.0 ** -140)


def close(got, want, tol):
    """got within tol of want, NaN where want is NaN, infinities alike; got in the type whose rounding is added to tol."""
    tol = tol + rounded(want, got.dtype)
    # a number past the type's range rounds to infinity: f32 ends at 3.4e38, and 1 / rms of rows of 1e-43 is 4e42
    past = want.to(got.dtype).double()
    got = got.cpu().double()
    assert got.shape == want.shape
    most = torch.finfo(torch.float64).max
    off = (got - want).abs()
    fine = (off <= tol) | (got.isnan() & want.isnan()) | (got == want) | (got.isinf() & (got == past))
    assert bool(fine.all()), (int((~fine).sum()), (off - tol).nan_to_num(most).max(), got[~fine][:4], want[~fine][:4])
