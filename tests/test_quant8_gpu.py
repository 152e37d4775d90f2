"""8-bit rows on the GPU against 64-bit arithmetic: the quantiser bit for bit, products and gated products within the
rounding of the scales and of the output."""
import math

import pytest
import torch

from scratchtape_amd import quant8
import quant8_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check_quantised(x, codes, scales, values=None):
    want, a = oracle.quantise(x.cpu().double())
    assert codes.dtype == torch.int8 and torch.equal(codes.cpu().long(), want)
    assert torch.equal(scales.cpu().nan_to_num(-1.0), (a / 127).float().nan_to_num(-1.0))
    if values is not None:
        assert values.dtype == x.dtype
        most = torch.finfo(x.dtype).max  # 127 f32(a / 127) can pass it
        exact = (want * scales.cpu().double()[:, None]).clamp(-most, most)
        oracle.close(values, exact, oracle.U * exact.abs() + 2.0 ** -149)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,k", [(1, 1), (1, 7), (3, 8), (5, 15), (7, 16), (9, 17), (33, 255), (4, 512), (6, 513), (5, 1023), (5, 1025), (130, 2048),
                                 (3, 2055), (3, 4097), (2, 8192), (2, 8201), (2, 16384), (3, 16391), (1, 40000), (768, 256)])
def test_quantiser_is_exact(dev, n, k, t):
    x = torch.randn(n, k, generator=gen(n + k)).to(TYPES[t]).to(dev)
    check_quantised(x, *quant8.quantize_8bit(x, values=True))
    codes, scales = quant8.quantize_8bit(x)
    check_quantised(x, codes, scales)
    assert codes.stride(0) % 16 == 0 or n == 1
    rows = codes.as_strided((n, (k + 15) // 16 * 16), ((k + 15) // 16 * 16, 1)).cpu()
    assert not rows[:, k:].any()  # zeros behind the rows' ends


@pytest.mark.parametrize("t", sorted(TYPES))
def test_quantiser_on_borders_and_extremes(dev, t):
    """Lattices of half steps (every border a tie), equal values, zeros, the type's range, subnormals, NaN and infinities."""
    t = TYPES[t]
    big, tiny = torch.finfo(t).max, torch.finfo(t).smallest_normal * torch.finfo(t).eps
    half = torch.arange(255) * 0.5  # up to 127: 0.5, 1.5 .. are ties
    rows = [half, -half, half * 2.0 ** -6, torch.full((255,), -3.25), torch.zeros(255), -torch.zeros(255),
            torch.tensor([1.0] + 254 * [0.0]), torch.linspace(-1, 1, 255) * big, torch.tensor([big, -big] + 253 * [1.0]),
            torch.arange(255) * tiny, torch.tensor([tiny] + 254 * [0.0]), torch.tensor([math.nan] + 254 * [1.0]),
            torch.tensor(254 * [2.0] + [math.inf]), torch.tensor([-math.inf, math.inf, math.nan] + 252 * [0.0]),
            torch.tensor([127.0, 0.5, 1.5, -2.5, 63.5] + 250 * [-126.5])]
    x = torch.stack([r.double().to(t) for r in rows]).to(dev)
    check_quantised(x, *quant8.quantize_8bit(x, values=True))
    y = torch.cat((x, x[:, :200]), 1).repeat(1, 3).contiguous()
    check_quantised(y, *quant8.quantize_8bit(y, values=True))


def test_quantiser_over_all_sizes_of_numbers(dev):
    """Rows from f32's subnormals to its largest values, quotients next to borders among them."""
    scale = torch.tensor([2.0 ** e for e in range(-149, 127)], dtype=torch.float64)[:, None]
    x = (torch.rand(276, 700, generator=gen(3), dtype=torch.float64) * 2 - 1) * scale
    x[:, 0] = scale[:, 0]
    x[:, 1:200] = (torch.arange(199) + 0.5)[None] / 127 * scale * 0.5  # borders of the codes, to f32
    check_quantised(x.float().to(dev), *quant8.quantize_8bit(x.float().to(dev), values=True))


@pytest.mark.parametrize("t", sorted(TYPES))
def test_quantiser_takes_views_and_fills_tensors(dev, t):
    base = torch.randn(9, 331, generator=gen(5)).to(TYPES[t]).to(dev)
    for view in (base[:, 3:260], base[::2, 8:264], base[1:2, 1:66], base[:, 330:]):
        out = torch.full(view.shape, 7.0, dtype=TYPES[t], device=dev)
        codes, scales, values = quant8.quantize_8bit(view, values=out)
        assert values is out
        check_quantised(view, codes, scales, values)
    codes, scales = quant8.quantize_8bit(base[:0])
    assert codes.shape == (0, 331) and scales.shape == (0,)


def operands(m, k, n, seed, dev):
    g = gen(seed)
    x = quant8.empty_codes(m, k, dev)
    w = quant8.empty_codes(n, k, dev)
    for c, rows in ((x, m), (w, n)):
        c.copy_(torch.randint(-127, 128, (rows, k), generator=g))
        if k % 16 and rows:  # what lies behind a row's end counts for nothing
            width = (k + 15) // 16 * 16
            c.as_strided((rows, width - k), (width, 1), k).fill_(77)
    xs, ws = torch.rand(m, generator=g) * 0.01, torch.rand(n, generator=g) * 0.001
    return x, xs.to(dev), w, ws.to(dev)


def check_product(ops, bias, relu, got):
    y, tol = oracle.product(*ops, bias)
    if relu:
        y = torch.where(y < 0, torch.zeros_like(y), y)
    oracle.close(got, y, tol)


# Rows of x from one token to more than two tiles, k and n around every power of two and tile
SHAPES = [(1, 1, 1), (1, 16, 1), (1, 64, 33), (1, 256, 1024), (1, 4096, 130), (2, 100, 70), (3, 31, 257), (8, 128, 64), (15, 129, 65), (16, 2048, 300),
          (17, 1000, 31), (31, 48, 129), (32, 512, 96), (33, 33, 33), (48, 4096, 515), (63, 127, 64), (64, 640, 128), (65, 64, 63), (97, 1280, 190),
          (127, 383, 255), (128, 128, 128), (129, 256, 257), (200, 1024, 320), (255, 96, 513), (256, 384, 256), (257, 4100, 384), (300, 2049, 511),
          (512, 512, 512), (515, 260, 1030), (1024, 256, 768)]


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product(dev, m, k, n):
    ops = operands(m, k, n, m + k + n, dev)
    bias = torch.randn(n, generator=gen(m)).to(dev)
    names = sorted(TYPES)
    t = TYPES[names[(m + n) % 3]]
    check_product(ops, None, False, quant8.matmul_8bit(*ops, dtype=t))
    check_product(ops, bias, True, quant8.matmul_8bit(*ops, bias=bias, relu=True, dtype=torch.float32))
    check_product(ops, bias, False, quant8.matmul_8bit(*ops, bias=bias, dtype=TYPES[names[(m + n + 1) % 3]]))


@pytest.mark.parametrize("m,k,n,activation", [(*s, a) for s in SHAPES for a in ("silu", "gelu") if a == "silu" or s[0] * s[2] <= 70000])
def test_gated_product(dev, m, k, n, activation):
    x, xs, w, ws = operands(m, k, 2 * n, m + k + n, dev)
    ws = ws * (200 / k ** 0.5)
    bias = torch.randn(2 * n, generator=gen(m)).to(dev)
    for t, b in ((TYPES[sorted(TYPES)[(m + n) % 3]], None), (torch.float32, bias)):
        y, tol = oracle.product(x, xs, w, ws, b)
        want, off = oracle.gated((y[:, :n], tol[:, :n]), (y[:, n:], tol[:, n:]), activation)
        oracle.close(quant8.gated_8bit(x, xs, w, ws, bias=b, activation=activation, dtype=t), want, off)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_product_of_strided_and_unaligned_rows(dev, t):
    """Rows 16 bytes apart or not, bases aligned or not, out with a stride, the columns beside it left alone."""
    g = gen(11)
    base_x = torch.randint(-127, 128, (300, 700), generator=g, dtype=torch.int8).to(dev)
    base_w = torch.randint(-127, 128, (420, 704), generator=g, dtype=torch.int8).to(dev)
    for rows, width in ((300, 333), (40, 640), (1, 257), (7, 16)):
        for off in (0, 1, 16, 20):
            x, w = base_x[:rows, off:off + width], base_w[::2, off:off + width]
            ops = (x, torch.rand(rows, generator=g).to(dev), w, torch.rand(210, generator=g).to(dev))
            out = torch.full((rows, 250), -3.0, dtype=TYPES[t], device=dev)
            scale = 1 / 4096
            ops = (ops[0], ops[1] * scale, ops[2], ops[3])
            got = quant8.matmul_8bit(*ops, dtype=TYPES[t], out=out[:, 17:227])
            check_product(ops, None, False, got)
            assert bool((out[:, :17] == -3).all()) and bool((out[:, 227:] == -3).all())


def test_extreme_sums(dev):
    """Sums at the ends of 32-bit integers: k = 131072 and codes of 127, and -128 beside 127."""
    k = 131072
    x = torch.full((33, k), 127, dtype=torch.int8, device=dev)
    w = torch.full((40, k), 127, dtype=torch.int8, device=dev)
    w[1::2] = -128
    x[2] = -127
    ones = torch.ones(40, device=dev)
    check_product((x, ones[:33], w, ones), None, False, quant8.matmul_8bit(x, ones[:33], w, ones, dtype=torch.float32))


def test_rows_that_are_not_finite_and_zero_rows(dev):
    """A row or channel of scale NaN is NaN throughout and leaves the others alone; zeros give the bias."""
    for m, k, n in ((4, 64, 40), (70, 256, 300), (300, 512, 300)):
        x, xs, w, ws = operands(m, k, n, 5, dev)
        xs[1], ws[3], xs[2], ws[5] = math.nan, math.nan, 0.0, 0.0
        bias = torch.randn(n, generator=gen(1)).to(dev)
        got = quant8.matmul_8bit(x, xs, w, ws, bias=bias, dtype=torch.float32).cpu()
        bad = torch.zeros(m, n, dtype=torch.bool)
        bad[1], bad[:, 3] = True, True
        assert torch.equal(got.isnan(), bad)
        check_product((x, xs, w, ws), bias, False, got)
        got = quant8.matmul_8bit(x, xs, w, ws, bias=bias, relu=True, dtype=torch.float32).cpu()
        assert torch.equal(got.isnan(), bad)


def test_nothing_to_do(dev):
    x, xs, w, ws = operands(0, 64, 5, 1, dev)
    assert quant8.matmul_8bit(x, xs, w, ws).shape == (0, 5)
    assert quant8.gated_8bit(x, xs, w[:4], ws[:4]).shape == (0, 2)
    x, xs, w, ws = operands(3, 64, 0, 1, dev)
    assert quant8.matmul_8bit(x, xs, w, ws).shape == (3, 0)


@pytest.mark.parametrize("m,k,n", [(1, 8192, 512), (48, 4096, 700), (300, 2048, 1000)])
def test_streams_and_graphs(dev, m, k, n):
    """Another stream, and a captured call replayed with eager work between, give the eager call's bits."""
    ops = operands(m, k, n, 9, dev)
    want = quant8.matmul_8bit(*ops, dtype=torch.float32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = quant8.matmul_8bit(*ops, dtype=torch.float32, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = quant8.matmul_8bit(*ops, dtype=torch.float32)
        y, ys = quant8.quantize_8bit(out)
        both = quant8.gated_8bit(ops[0], ops[1], ops[2][:n // 2 * 2], ops[3][:n // 2 * 2], dtype=torch.float32)
    eager = quant8.gated_8bit(ops[0], ops[1], ops[2][:n // 2 * 2], ops[3][:n // 2 * 2], dtype=torch.float32)
    codes, scales = quant8.quantize_8bit(want)
    for i in range(3):
        out.zero_(), both.zero_()
        graph.replay()
        assert torch.equal(quant8.matmul_8bit(*ops, dtype=torch.float32), want)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(y, codes) and torch.equal(ys, scales) and torch.equal(both, eager)
