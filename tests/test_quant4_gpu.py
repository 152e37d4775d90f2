"""4-bit weights on the GPU against 64-bit arithmetic: the quantiser bit for bit, the products within the error that f32
sums over exact products allow."""
import math

import pytest
import torch

from scratchtape_amd import quant4
import quant4_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def weights(n, k, t, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, k, generator=g) * spread).to(t)


def check_quantised(x, group, codes, scales, values=None):
    n, k = x.shape
    want, scale, lo = oracle.quantise(x.cpu().unflatten(-1, (-1, group)))
    assert torch.equal(codes.cpu(), oracle.pack(want).reshape(n, k // 2))
    got = scales.cpu().double()
    assert torch.equal(got[..., 0].nan_to_num(-1), scale[..., 0].nan_to_num(-1))
    assert torch.equal(got[..., 1].nan_to_num(-1), lo[..., 0].nan_to_num(-1))
    if values is not None:
        exact = want * scale + lo
        # one rounding to the type, and a product and a sum in f32
        tol = torch.finfo(x.dtype).eps / 2 * exact.abs() + 2.0 ** -23 * (want * scale + lo.abs()) + 2.0 ** -133
        if x.dtype == torch.float16:
            tol = tol + 2.0 ** -25
        off = (values.cpu().double().unflatten(-1, (-1, group)) - exact).abs()
        assert bool(((off <= tol) | (off.isnan() & exact.isnan())).all()), (off - tol).max()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (1, 128, 128), (3, 64, 64), (7, 96, 32), (33, 192, 64), (129, 1152, 128),
                                       (768, 256, 64), (5, 8192, 32)])
def test_quantiser_is_exact(dev, n, k, group, t):
    x = weights(n, k, TYPES[t], n + k).to(dev)
    check_quantised(x, group, *quant4.quantize_4bit(x, group, values=True))
    codes, scales = quant4.quantize_4bit(x, group)
    check_quantised(x, group, codes, scales)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_quantiser_on_borders_ties_and_extremes(dev, t):
    """Values on the borders of two codes (a lattice of half steps), equal values, one value alone, the type's range, values
    next to nothing, signed zeros, and groups that hold a NaN or an infinity."""
    t = TYPES[t]
    big = torch.finfo(t).max / 4
    lattice = torch.arange(32).remainder(31) * 0.5  # 0, 0.5 .. 15: every border is a tie
    rows = [lattice, -lattice, lattice * 2.0 ** -12, torch.full((32,), 3.25), torch.zeros(32),
            torch.cat((torch.zeros(16), -torch.zeros(16))), torch.tensor([1.0] + 31 * [0.0]),
            torch.linspace(-1, 1, 32) * big, torch.tensor([big, -big] + 30 * [1.0]),
            torch.arange(32) * torch.finfo(t).smallest_normal * torch.finfo(t).eps,
            torch.tensor([math.nan] + 31 * [1.0]), torch.tensor(31 * [2.0] + [math.inf]), torch.tensor([-math.inf, math.inf] + 30 * [0.0]),
            1000 + torch.arange(32) / 16, torch.tensor([1e4] + 31 * [1e-4])]
    x = torch.stack([r.double().to(t) for r in rows]).to(dev)
    check_quantised(x, 32, *quant4.quantize_4bit(x, 32, values=True))
    y = x.repeat(1, 4).contiguous()
    for group in (64, 128):
        check_quantised(y, group, *quant4.quantize_4bit(y, group, values=True))


def test_quantiser_over_all_sizes_of_numbers(dev):
    """Group widths from f32's subnormals to its largest values, each far from zero and near it: the quotients in f32 and those
    in 64 bits hold the same codes."""
    g = torch.Generator().manual_seed(21)
    scale = torch.tensor([2.0 ** e for e in range(-146, 126)], dtype=torch.float64)[:, None]
    x = torch.rand(272, 1024, generator=g, dtype=torch.float64) * scale
    x = torch.cat((x, x + 3 * scale, x - 2 * scale)).float().to(dev)
    for group in (32, 128):
        check_quantised(x, group, *quant4.quantize_4bit(x, group, values=True))


def test_quantiser_of_short_and_of_strided_rows(dev):
    """Rows shorter than a workgroup's share, apart and together."""
    for n, k, stride in ((1000, 32, 35), (77, 96, 96), (513, 64, 64), (3, 8192, 8200), (5, 2080, 2084)):
        x = weights(n, stride, torch.float32, n).to(dev)[:, :k]
        check_quantised(x, 32, *quant4.quantize_4bit(x, 32, values=True))


@pytest.mark.parametrize("t", sorted(TYPES))
def test_quantiser_takes_views_and_fills_tensors(dev, t):
    base = weights(9, 331, TYPES[t], 5).to(dev)
    for view in (base[:, 3:3 + 256], base[::2, 8:264], base[1:2, 1:65]):
        n, k = view.shape
        out = torch.full((n, k), 7.0, dtype=TYPES[t], device=dev)
        codes, scales, values = quant4.quantize_4bit(view, 64, values=out)
        assert values is out
        check_quantised(view, 64, codes, scales, values)
    codes, scales = quant4.quantize_4bit(base[:0, :64], 64)
    assert codes.shape == (0, 32) and scales.shape == (0, 1, 2)


def product(x, codes, scales, bias, relu):
    """The product in 64 bits and how far an output may be off."""
    m, k = x.shape
    n, groups = scales.shape[:2]
    c = oracle.unpack(codes.cpu()).view(n, groups, -1)
    s = scales.cpu().double()
    w = (c * s[..., :1] + s[..., 1:]).view(n, k)
    w_abs = (c * s[..., :1] + s[..., 1:].abs()).view(n, k)
    xd = x.cpu().double()
    y = xd @ w.t()
    size = xd.abs() @ w_abs.t()
    if bias is not None:
        y, size = y + bias.cpu().double(), size + bias.cpu().double().abs()
    if relu:
        y = y.clamp(min=0)
    # f32 sums of exact products in any order with chains of k / 32 + 64 additions at most; f32 rows to 22 bits
    tol = (64 + k / 32) * 2.0 ** -24 * size + torch.finfo(x.dtype).eps / 2 * y.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    return y, tol


def check_product(x, codes, scales, bias, relu, got):
    y, tol = product(x, codes, scales, bias, relu)
    got = got.cpu().double()
    off = (got - y).abs()
    # Beyond its largest value a type's nearest is infinity: from half a step past it on (f16: 65504 + 16), less the error.
    big = torch.finfo(x.dtype).max * (1 + torch.finfo(x.dtype).eps / 4)
    past = got.isinf() & (got.sign() == y.sign()) & (y.abs() + tol >= big)
    assert bool(((off <= tol) | past).all()), (off / tol)[~past].max()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("m,k,n,group", [(1, 32, 1, 32), (1, 256, 1024, 64), (1, 8192, 77, 128), (2, 96, 17, 32), (3, 192, 130, 64),
                                         (16, 4096, 515, 32), (17, 640, 255, 128), (33, 1088, 64, 64), (70, 128, 300, 128),
                                         (1, 20480, 16, 32), (5, 32, 40000, 32), (16, 1056, 8200, 32), (20, 640, 8200, 64),
                                         (2, 1408, 8255, 128)])
def test_products_against_64_bits(dev, m, k, n, group, t):
    g = torch.Generator().manual_seed(m + k + n)
    codes, scales = quant4.quantize_4bit(torch.randn(n, k, generator=g).to(dev) * 0.05, group)
    x = torch.randn(m, k, generator=g).to(TYPES[t]).to(dev)
    bias = torch.randn(n, generator=g).to(dev)
    check_product(x, codes, scales, None, False, quant4.matvec_4bit(x, codes, scales))
    check_product(x, codes, scales, bias, True, quant4.matvec_4bit(x, codes, scales, bias=bias, relu=True))


@pytest.mark.parametrize("t", sorted(TYPES))
def test_products_of_views_scales_and_magnitudes(dev, t):
    """Rows and outputs at odd strides; rows of very different sizes in one call; weights with offsets far from zero; the rest
    of the output's memory untouched."""
    t = TYPES[t]
    g = torch.Generator().manual_seed(3)
    n, k = 203, 384
    codes, scales = quant4.quantize_4bit((torch.randn(n, k, generator=g) * 0.01 + 3.0).to(dev), 64)
    base = torch.randn(6, 401, generator=g)
    base *= torch.tensor([1.0, 1e-4, 1e3, 0.0, 1e-2, 7.0])[:, None]
    base = base.to(t).to(dev)
    store = torch.full((6, 211), 5.0, dtype=t, device=dev)
    for shift in (0, 1, 8):
        x, out = base[:, shift:shift + k], store[:, 2:2 + n]
        assert quant4.matvec_4bit(x, codes, scales, out=out) is out
        check_product(x, codes, scales, None, False, out)
        assert bool((store[:, :2] == 5).all()) and bool((store[:, 2 + n:] == 5).all())
    assert quant4.matvec_4bit(base[:0, :k], codes, scales).shape == (0, n)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_products_with_values_that_are_not_finite(dev, t):
    """A NaN or infinite input spoils its own row alone; a NaN weight group its own column alone."""
    t = TYPES[t]
    g = torch.Generator().manual_seed(4)
    w = torch.randn(50, 256, generator=g)
    w[7, 40] = math.nan
    codes, scales = quant4.quantize_4bit(w.to(dev), 32)
    x = torch.randn(5, 256, generator=g).to(t)
    x[1, 3], x[3, 200] = math.inf, math.nan
    y = quant4.matvec_4bit(x.to(dev), codes, scales).cpu()
    bad = torch.zeros(5, 50, dtype=torch.bool)
    bad[:, 7] = True
    assert bool(y[:, 7].isnan().all()) and bool(y[3].isnan().all())
    assert not bool(torch.isfinite(y[1]).any())
    clean = x.clone()
    clean[[1, 3]] = 0
    good = quant4.matvec_4bit(clean.to(dev), codes, scales).cpu()
    assert torch.equal(y[[0, 2, 4]].nan_to_num(9), good[[0, 2, 4]].nan_to_num(9)) and bool(torch.isfinite(good[:, :7]).all())
    # (Fewer rows may be summed in another order: those are held to the exact products, not to the bits above.)
    few, rest = x[[0, 2, 4]].contiguous(), [i for i in range(50) if i != 7]
    y = quant4.matvec_4bit(few.to(dev), codes, scales)
    check_product(few.to(dev), codes[rest], scales[rest], None, False, y[:, rest])
    assert bool(y[:, 7].isnan().all())


def test_weights_past_4_gib(dev):
    """Codes of more than 2^32 bytes: the last rows of a 2,200,000 x 4096 weight."""
    n, k = 2_200_000, 4096
    codes = torch.empty(n, k // 2, dtype=torch.uint8, device=dev)
    scales = torch.zeros(n, k // 128, 2, device=dev)
    codes.fill_(0x21)
    g = torch.Generator().manual_seed(8)
    tail, tail_scales = quant4.quantize_4bit(torch.randn(64, k, generator=g).to(dev), 128)
    codes[-64:], scales[-64:] = tail, tail_scales
    x = torch.randn(1, k, generator=g).to(dev)
    y = quant4.matvec_4bit(x, codes, scales)
    check_product(x, tail, tail_scales, None, False, y[:, -64:])
    assert not bool(y[:, :-64].any())


def test_another_stream_and_a_captured_graph(dev):
    g = torch.Generator().manual_seed(9)
    w, x = torch.randn(640, 512, generator=g).to(dev), torch.randn(4, 512, generator=g).to(dev)
    codes, scales = quant4.quantize_4bit(w, 64)
    want = quant4.matvec_4bit(x, codes, scales)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    c2, s2 = quant4.quantize_4bit(w, 64, stream=side)
    y2 = quant4.matvec_4bit(x, c2, s2, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(c2, codes) and torch.equal(s2, scales) and torch.equal(y2, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c3, s3 = quant4.quantize_4bit(w, 64)
        y3 = quant4.matvec_4bit(x, c3, s3, relu=True)
    for i in range(3):
        w.copy_(torch.randn(640, 512, generator=g))
        x.copy_(torch.randn(4, 512, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        ce, se = quant4.quantize_4bit(w, 64)
        assert torch.equal(c3, ce) and torch.equal(s3, se)
        assert torch.equal(y3, quant4.matvec_4bit(x, ce, se, relu=True))
