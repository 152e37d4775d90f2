"""8-bit products whose workgroups take several tiles one after the other, on each of the kernels, at sizes that divide and
that do not, against 64-bit products on the GPU."""
import pytest
import torch

from scratchtape_amd import quant8
import quant8_oracle as oracle

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def operands(m, k, n, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    made = []
    for rows in (m, n):
        codes = quant8.empty_codes(rows, k, dev)
        codes.copy_(torch.randint(-127, 128, (rows, k), generator=g, device=dev, dtype=torch.int8))
        made += [codes, torch.rand(rows, generator=g, device=dev) * 0.02]
    return made


def close(got, want, tol):
    """oracle.close on the GPU: the sizes here are too large to bring over."""
    rel, tiny = oracle.half_step(got.dtype)
    off = (got.double() - want).abs()
    bad = ~(off <= tol + rel * want.abs() + tiny)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4], want[bad][:4])


def product(x, xs, w, ws, bias):
    s = torch.matmul(x.double(), w.double().t()) * xs.double()[:, None] * ws.double()
    y = s if bias is None else s + bias.double()
    return y, 2.01 * oracle.U * s.abs() + oracle.U * y.abs() + 2.0 ** -148


LINEAR = [("large", 8192, 1024, 8192, BF16), ("large", 4100, 2085, 8200, F32), ("large", 2300, 4096, 11000, F16), ("large", 16000, 64 * 17, 3000, F32),
          ("middle", 8192, 512, 8192, F32), ("middle", 8200, 333, 8195, BF16), ("middle", 700, 16, 20000, F16), ("middle", 3000, 100, 5001, F32),
          ("small", 1000, 128, 1000, F32), ("small", 300, 1000, 1500, BF16), ("small", 129, 4100, 4099, F32), ("small", 200, 16384, 500, F16),
          ("small", 100, 131072, 70, F32), ("deep", 64, 256, 40000, F32), ("deep", 33, 4096, 515, BF16), ("deep", 48, 4096, 11003, F16),
          ("deep", 5, 131072, 33, F32), ("deep", 17, 4111, 30000, F32), ("deep", 64, 16384, 1024, BF16), ("few", 20, 300, 3001, F32), ("few", 7, 2050, 40, F16),
          ("one", 3, 1000, 50000, F32), ("one", 1, 65536, 300, BF16), ("one", 2, 8200, 5000, F16), ("one", 4, 16384, 7, F32)]


@pytest.mark.parametrize("kernel,m,k,n,t", LINEAR)
def test_product(dev, kernel, m, k, n, t):
    assert quant8.product_plan(m, k, n)[0] == kernel
    ops = operands(m, k, n, m + n, dev)
    bias = torch.randn(n, generator=torch.Generator(device=dev).manual_seed(n), device=dev)
    ops[1] *= 20 / k ** 0.5 / 100  # within f16's range
    for b, relu in ((None, False), (bias, True)):
        y, tol = product(*ops, b)
        close(quant8.matmul_8bit(*ops, bias=b, relu=relu, dtype=t), y.clamp(min=0) if relu else y, tol)


GATED = [("large", 4096, 2048, 8192, BF16), ("large", 2050, 1100, 10000, F16), ("large", 1000, 4096, 12300, F32), ("middle", 700, 512, 20000, F32),
         ("middle", 130, 4096, 12288, F16), ("low", 200, 1024, 1024, F32), ("low", 90, 333, 6001, BF16), ("deep_low", 40, 512, 20000, F32),
         ("deep_low", 64, 2085, 8200, F16), ("deep_low", 16, 4096, 12288, BF16), ("few", 7, 2048, 300, F32), ("few", 30, 500, 700, F16), ("one", 4, 3000, 3001, F32),
         ("one", 1, 8192, 4000, BF16)]


@pytest.mark.parametrize("kernel,m,k,n,t", GATED)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gated_product(dev, kernel, m, k, n, t, activation):
    assert quant8.product_plan(m, k, n, gated=True)[0] == kernel
    x, xs, w, ws = operands(m, k, 2 * n, m + n, dev)
    xs *= 4 / k ** 0.5 / 100
    y, tol = product(x, xs, w, ws, None)
    want, off = oracle.gated((y[:, :n], tol[:, :n]), (y[:, n:], tol[:, n:]), activation)
    close(quant8.gated_8bit(x, xs, w, ws, activation=activation, dtype=t), want, off)


SLICED = [s for s in ((100, 8192, 60), (200, 16384, 100), (33, 16384, 100), (64, 131072, 40), (70, 5000, 130))]


@pytest.mark.parametrize("m,k,n", SLICED)
def test_gated_product_in_slices(dev, m, k, n):
    assert quant8.product_plan(m, k, n, gated=True)[1] > 1
    x, xs, w, ws = operands(m, k, 2 * n, m + n, dev)
    xs *= 4 / k ** 0.5 / 100
    y, tol = product(x, xs, w, ws, None)
    want, off = oracle.gated((y[:, :n], tol[:, :n]), (y[:, n:], tol[:, n:]), "gelu")
    close(quant8.gated_8bit(x, xs, w, ws, activation="gelu", dtype=F32), want, off)


@pytest.mark.parametrize("m,k,n", [(4100, 2085, 8200), (8200, 333, 8195), (1000, 128, 3000), (64, 256, 40000), (48, 16384, 515), (20, 300, 3001), (3, 1000, 50000)])
def test_nothing_is_written_beside_the_output(dev, m, k, n):
    """Rows of out a stride apart: what lies between them, before and behind stays; a second call gives the same bits."""
    ops = operands(m, k, n, 3, dev)
    for t in (F32, BF16):
        whole = torch.full((m + 2, n + 24), -7.0, dtype=t, device=dev)
        out = whole[1:m + 1, 8:n + 8]
        got = quant8.matmul_8bit(*ops, dtype=t, out=out)
        assert got is out
        assert torch.equal(out, quant8.matmul_8bit(*ops, dtype=t))
        out.fill_(-7.0)
        assert bool((whole == -7).all())


def test_unaligned_rows_give_the_same_bits(dev):
    """Codes a byte off their alignment take the kernel for any strides."""
    for m, k, n in ((300, 512, 700), (5, 1000, 64), (1, 4096, 130)):
        x, xs, w, ws = operands(m, k, n, 9, dev)
        off = torch.empty(m * (k + 1) + 1, dtype=torch.int8, device=dev)[1:].view(m, k + 1)[:, :k]
        off.copy_(x)
        assert off.data_ptr() % 16 == 1 or m == 1
        assert torch.equal(quant8.matmul_8bit(off, xs, w, ws, dtype=F32), quant8.matmul_8bit(x, xs, w, ws, dtype=F32))
        half = n // 2 * 2
        assert torch.equal(quant8.gated_8bit(off, xs, w[:half], ws[:half], dtype=F32), quant8.gated_8bit(x, xs, w[:half], ws[:half], dtype=F32))


def test_two_streams_at_once(dev):
    """Two calls in slices at the same time have work memory of their own."""
    ops = operands(64, 16384, 1024, 4, dev), operands(200, 16384, 500, 5, dev)
    assert all(quant8.product_plan(m, 16384, n)[1] > 1 for m, n in ((64, 1024), (200, 500)))
    want = [quant8.matmul_8bit(*o, dtype=F32) for o in ops]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ops]
    for _ in range(5):
        got = [quant8.matmul_8bit(*o, dtype=F32, stream=s) for o, s in zip(ops, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
