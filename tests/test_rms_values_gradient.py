"""Training through the values of 8-bit rows (the straight-through form): the norm's rstd without a y that nobody reads."""
import pytest
import torch

from scratchtape_amd import rows
import quant8_oracle as oracle


def test_rstd_alone_is_refused():
    x = torch.zeros(4, 96)
    with pytest.raises(ValueError, match="neither"):
        rows.rms_norm(x, torch.ones(96), y=False, rstd=True)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(1, 1), (5, 300), (128, 256), (40, 2051), (3, 8192), (2, 17000)])
def test_gradient_through_values(dev, n, d, t):
    g = torch.Generator().manual_seed(n + d)
    x, r, dv = (torch.randn(n, d, generator=g).to(t).to(dev) for _ in range(3))
    w = (1 + 0.3 * torch.randn(d, generator=g)).to(dev)
    with_y = rows.rms_norm(x, w, residual=r, eight_bit=True, values=True)
    out = rows.rms_norm(x, w, residual=r, y=False, eight_bit=True, values=True, rstd=True)
    assert out.y is None and torch.equal(out.rstd, with_y.rstd) and torch.equal(out.values, with_y.values) and torch.equal(out.codes, with_y.codes)
    assert rows.rms_norm(x, w, y=False, eight_bit=True).rstd is None
    oracle.close(out.rstd, oracle.norm(x, r, w, 1e-5)[1], 2.0 ** -50 * out.rstd.cpu().double())
    dx, dw = rows.rms_norm_backward(dv, out.h, out.rstd, w)
    (ex, tx), (ew, tw) = oracle.norm_backward(dv, out.h, out.rstd, w, None)
    oracle.close(dx, ex, tx)
    oracle.close(dw, ew, tw)
