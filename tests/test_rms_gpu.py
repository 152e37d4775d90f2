"""The root-mean-square norm, its 8-bit rows and its gradients on the GPU against 64-bit arithmetic."""
import math

import pytest
import torch

from scratchtape_amd import rows
import quant8_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(1, 1), (1, 8), (3, 7), (5, 17), (128, 256), (9, 500), (4, 512), (7, 513), (6, 1000), (5, 1024), (3, 1025), (33, 2048), (2, 2051), (3, 4096),
          (2, 4099), (5, 8192), (2, 8200), (3, 16384), (2, 16390), (1, 50001)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def inputs(n, d, t, wt, seed, dev):
    g = gen(seed)
    make = lambda *s: torch.randn(*s, generator=g)
    return make(n, d).to(t).to(dev), make(n, d).mul(3).to(t).to(dev), (1 + 0.3 * make(d)).to(wt).to(dev)


def check(x, residual, w, eps, out, y=True, eight=False, values=False):
    h, rstd, want, t = oracle.norm(x, residual, w, eps)
    assert torch.equal(out.h.cpu().nan_to_num(77), h.nan_to_num(77))
    if y:
        oracle.close(out.rstd, rstd, 2.0 ** -50 * rstd)
        oracle.close(out.y, want, oracle.U * want.abs() + 2.0 ** -149)
    if eight:
        codes, a = oracle.quantise(t)
        assert torch.equal(out.codes.cpu().long(), codes)
        scale = a * rstd / 127
        oracle.close(out.scales, scale, 2.0 ** -50 * scale)
        if values:
            most = torch.finfo(x.dtype).max
            exact = (codes * out.scales.cpu().double()[:, None]).clamp(-most, most)
            oracle.close(out.values, exact, oracle.U * exact.abs() + 2.0 ** -149)
    assert (out.y is not None) == (out.rstd is not None) == y and (out.codes is not None) == eight and (out.values is not None) == values


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,d", SHAPES)
def test_norm(dev, n, d, t):
    t = TYPES[t]
    for wt in {t, torch.float32}:
        x, r, w = inputs(n, d, t, wt, n + d, dev)
        check(x, r, w, 1e-5, rows.rms_norm(x, w, residual=r))
        check(x, None, w, 1e-6, rows.rms_norm(x, w, eps=1e-6, eight_bit=True), eight=True)
        out = rows.rms_norm(x, w, residual=r, eps=0.0, y=False, eight_bit=True, values=True)
        check(x, r, w, 0.0, out, y=False, eight=True, values=True)
        padded = out.codes.as_strided((n, (d + 15) // 16 * 16), ((d + 15) // 16 * 16, 1)).cpu()
        assert not padded[:, d:].any()


@pytest.mark.parametrize("t", sorted(TYPES))
def test_norm_of_extreme_rows(dev, t):
    """Zeros, the type's largest and smallest values (squares past f32's range), NaN and infinities, sums that overflow the
    type: each row by itself."""
    t = TYPES[t]
    info = torch.finfo(t)
    d = 300
    rows_of = [torch.zeros(d), torch.full((d,), float(info.max)), torch.full((d,), float(info.smallest_normal)), torch.linspace(-1, 1, d) * float(info.max),
               torch.arange(d) * (float(info.smallest_normal) * info.eps), torch.tensor([math.nan] + (d - 1) * [1.0]),
               torch.tensor((d - 1) * [1.0] + [-math.inf]), torch.randn(d, generator=gen(1))]
    x = torch.stack([r.double().to(t) for r in rows_of]).to(dev)
    w = (1 + torch.rand(d, generator=gen(2))).to(t).to(dev)
    # The formula of a row with an infinity is NaN at the infinity and 0 elsewhere: rstd is 0.
    for eps in (1e-5, 0.0):
        finite = [0, 1, 2, 3, 4, 7] if eps else [1, 2, 3, 4, 7]
        out = rows.rms_norm(x, w, eps=eps, eight_bit=True)
        for i in finite:
            one = rows.RmsOut(out.h[i:i + 1], out.rstd[i:i + 1], out.y[i:i + 1], out.codes[i:i + 1], out.scales[i:i + 1])
            check(x[i:i + 1], None, w, eps, one, eight=True)
        for i in (5, 6):
            assert bool(out.scales[i].isnan()) and not out.codes[i].any()
        assert bool(out.y[5].isnan().all()) and bool(out.y[6, -1].isnan()) and not out.y[6, :-1].any()
    # a sum past the type's range is infinite, as the kept sum is
    big = torch.full((2, d), float(info.max) * 0.75).to(t).to(dev)
    big[1] = 1
    out = rows.rms_norm(big, w, residual=big, eight_bit=True)
    assert bool(out.h[0].isinf().all()) and bool(out.scales[0].isnan()) and not out.codes[0].any() and bool(out.y[0].isnan().all())
    check(big[1:], big[1:], w, 1e-5, rows.RmsOut(out.h[1:], out.rstd[1:], out.y[1:], out.codes[1:], out.scales[1:]), eight=True)


def test_codes_on_borders(dev):
    """Products h w on borders of two codes, to the last bit of 48: lattices with weights that are powers of two, and rows of f32
    whose products straddle borders."""
    d = 255
    h = (torch.arange(d) * 0.5).repeat(4, 1)
    w = 2.0 ** torch.randint(-3, 4, (d,), generator=gen(3)).float()
    h = h / w  # h w is the lattice of half steps
    x = h.to(dev)
    check(x, None, w.to(dev), 1e-5, rows.rms_norm(x, w.to(dev), eight_bit=True, values=True), eight=True, values=True)
    g = gen(8)
    w = 1 + torch.rand(d, generator=g)
    border = (torch.randint(0, 126, (64, d), generator=g).double() + 0.5) / 127 * 3.7
    h = (border / w.double()).float()
    h[:, 0] = 3.7 / w[0]
    x = h.to(dev)
    check(x, None, w.to(dev), 1e-5, rows.rms_norm(x, w.to(dev), eight_bit=True), eight=True)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_norm_of_views(dev, t):
    base = torch.randn(20, 1301, generator=gen(4)).to(TYPES[t]).to(dev)
    w = torch.rand(640, generator=gen(5)).to(dev)
    for x, r in ((base[:, 1:641], base[:, 643:1283]), (base[::2, :640], base[1::2, 661:1301]), (base[3:4, 7:647], base[9:10, 8:648])):
        check(x, r, w, 1e-5, rows.rms_norm(x, w, residual=r, eight_bit=True, values=True), eight=True, values=True)
        h = rows.rms_norm(x, w)
        dx, dw = rows.rms_norm_backward(r, x, h.rstd, w, dh=x)
        (ex, tx), (ew, tw) = oracle.norm_backward(r, x, h.rstd, w, x)
        oracle.close(dx, ex, tx)
        oracle.close(dw, ew, tw)
    out = rows.rms_norm(base[:0, :640], w, eight_bit=True)
    assert out.y.shape == (0, 640) and out.codes.shape == (0, 640) and out.rstd.shape == (0,)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,d", SHAPES + [(4096, 256), (1500, 64), (3000, 520), (2000, 1100), (1100, 3008), (70, 8192), (40, 10001), (100, 17000)])
def test_backward(dev, n, d, t):
    t = TYPES[t]
    for wt in {t, torch.float32}:
        x, dy, w = inputs(n, d, t, wt, n + d, dev)
        dh = torch.randn(n, d, generator=gen(7)).to(t).to(dev)
        rstd = rows.rms_norm(x, w).rstd
        for more in (None, dh):
            dx, dw = rows.rms_norm_backward(dy, x, rstd, w, dh=more)
            assert dx.dtype == t and dw.dtype == torch.float32
            (ex, tx), (ew, tw) = oracle.norm_backward(dy, x, rstd, w, more)
            oracle.close(dx, ex, tx)
            oracle.close(dw, ew, tw)


def test_backward_is_the_gradient(dev):
    """Against torch's differentiation of the formula in 64 bits, and against differences of the forward pass itself."""
    g = gen(12)
    x = torch.randn(6, 40, generator=g, dtype=torch.float64)
    r, w, dy, dh = torch.randn(6, 40, generator=g).double(), torch.rand(40, generator=g).double() + 0.5, torch.randn(6, 40, generator=g).double(), torch.randn(6, 40, generator=g).double()

    def loss(x, r, w):
        h = x + r
        return ((h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-3) * w) * dy).sum() + (h * dh).sum()

    leaves = [v.float().double().requires_grad_() for v in (x, r, w)]
    gx, gr, gw = torch.autograd.grad(loss(*leaves), leaves)
    assert torch.equal(gx, gr)
    f = [v.detach().float().to(dev) for v in leaves]
    out = rows.rms_norm(f[0], f[2], residual=f[1], eps=1e-3)
    dx, dw = rows.rms_norm_backward(dy.float().to(dev), out.h, out.rstd, f[2], dh=dh.float().to(dev))
    # f32 inputs of size 3 and less, sums of 40: the roundings of h, rstd and dy are 2^-24 each of terms up to about 30
    assert float((dx.cpu().double() - gx).abs().max()) < 40 * 2.0 ** -20 and float((dw.cpu().double() - gw).abs().max()) < 40 * 2.0 ** -20
    # differences of the f32 forward: y is good to 2^-24 of its size, so a step of 2^-8 leaves about 40 x 6 x 2^-24 x 2^8 = 2^-8
    step = 2.0 ** -8
    dyf, dhf = dy.float(), dh.float()
    for i, j in ((0, 0), (3, 17), (5, 39)):
        sides = []
        for s in (step, -step):
            moved = f[0].clone()
            moved[i, j] += s
            o = rows.rms_norm(moved, f[2], residual=f[1], eps=1e-3)
            sides.append(float((o.y.cpu().double() * dy).sum() + (o.h.cpu().double() * dhf.double()).sum()))
        assert abs((sides[0] - sides[1]) / (2 * step) - float(gx[i, j])) < 2.0 ** -6


def test_backward_without_rows(dev):
    x = torch.zeros(0, 96, device=dev)
    w = torch.ones(96, device=dev)
    dx, dw = rows.rms_norm_backward(x, x, torch.zeros(0, device=dev), w)
    assert dx.shape == (0, 96) and not dw.any()


def test_streams_and_graphs(dev):
    x, r, w = inputs(700, 1024, torch.bfloat16, torch.float32, 3, dev)
    want = rows.rms_norm(x, w, residual=r, eight_bit=True)
    grads = rows.rms_norm_backward(r, want.h, want.rstd, w, dh=x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = rows.rms_norm(x, w, residual=r, eight_bit=True, stream=s)
    back = rows.rms_norm_backward(r, got.h, got.rstd, w, dh=x, stream=s)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = rows.rms_norm(x, w, residual=r, eight_bit=True)
        kept_back = rows.rms_norm_backward(r, kept.h, kept.rstd, w, dh=x)
    for i in range(3):
        kept.y.zero_(), kept_back[1].zero_()
        graph.replay()
        assert torch.equal(rows.rms_norm_backward(r, want.h, want.rstd, w, dh=x)[0], grads[0])
        torch.cuda.synchronize()
        for a, b in ((got, want), (kept, want)):
            for name in ("h", "rstd", "y", "codes", "scales"):
                assert torch.equal(getattr(a, name), getattr(b, name)), name
        for a in (back, kept_back):
            assert torch.equal(a[0], grads[0]) and torch.equal(a[1], grads[1])


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("d", [*range(1, 16), *range(505, 512), *range(1097, 1104), *range(4001, 4008), *range(9001, 9008)])
def test_ends_of_rows(dev, d, t):
    """Every number of elements behind a row's last eight; rows apart, with NaN between them that nothing may read."""
    t = TYPES[t]
    w = (1 + 0.3 * torch.randn(d, generator=gen(d))).to(t).to(dev)

    def apart(seed):
        base = torch.full((6, d + 9), math.nan, dtype=t, device=dev)
        base[:, 5:5 + d] = torch.randn(6, d, generator=gen(seed)).to(t).to(dev)
        return base[:, 5:5 + d]

    x, r, dy, dh = (apart(s) for s in range(4))
    check(x, r, w, 1e-5, rows.rms_norm(x, w, residual=r, eight_bit=True, values=True), eight=True, values=True)
    rstd = rows.rms_norm(x, w).rstd
    for more in (None, dh):
        dx, dw = rows.rms_norm_backward(dy, x, rstd, w, dh=more)
        (ex, tx), (ew, tw) = oracle.norm_backward(dy, x, rstd, w, more)
        oracle.close(dx, ex, tx)
        oracle.close(dw, ew, tw)


def test_backward_of_one_long_row(dev):
    """A row so wide that the launch that joins the parts has more workgroups than fit one line of a grid."""
    d = (1 << 25) + 17
    x, dy = (torch.randn(33, d, generator=torch.Generator(dev).manual_seed(s), device=dev, dtype=torch.bfloat16) for s in (1, 2))
    w, rstd = torch.ones(d, device=dev), torch.ones(33, device=dev)
    dx, dw = rows.rms_norm_backward(dy, x, rstd, w)
    for part in (slice(0, 40), slice(d // 2, d // 2 + 40), slice(d - 40, d)):
        products = dy[:, part].cpu().double() * x[:, part].cpu().double()
        oracle.close(dw[part], products.sum(0), 40 * oracle.U * products.abs().sum(0))
