"""Operands of more than 2^32 bytes: rows past that offset give what the same rows give by themselves."""
import pytest
import torch

from scratchtape_amd import quant8, rows
import quant8_oracle as oracle

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
FAR = 525_003  # rows of 8192 bytes: the last 715 are past 2^32


def codes(n, k, seed, dev):
    g = torch.Generator(dev).manual_seed(seed)
    return (torch.randint(-127, 128, (n, k), dtype=torch.int8, generator=g, device=dev),
            torch.rand((n,), generator=g, device=dev) / (100 * k ** 0.5))


def test_weights_past_4_gb(dev):
    w, ws = codes(FAR, 8192, 1, dev)
    assert w.numel() > 1 << 32
    for m in (1, 8, 40, 300):
        x, xs = codes(m, 8192, 2, dev)
        got = quant8.matmul_8bit(x, xs, w, ws, dtype=F32)
        for part in (slice(0, 70), slice(FAR - 740, FAR)):
            assert torch.equal(got[:, part], quant8.matmul_8bit(x, xs, w[part], ws[part], dtype=F32))
        want, off = oracle.product(x, xs, w[-9:], ws[-9:])
        oracle.close(got[:, -9:], want, off)


def test_gated_weights_past_4_gb(dev):
    n = FAR // 2
    w, ws = codes(2 * n, 8192, 3, dev)
    for m in (1, 8, 70):
        x, xs = codes(m, 8192, 4, dev)
        got = quant8.gated_8bit(x, xs, w, ws, dtype=F32)
        for part in (slice(0, 70), slice(n - 740, n)):
            both = [torch.cat([t[:n][part], t[n:][part]]) for t in (w, ws)]
            assert torch.equal(got[:, part], quant8.gated_8bit(x, xs, *both, dtype=F32))


def test_rows_and_outputs_past_4_gb(dev):
    x, xs = codes(FAR, 8192, 5, dev)
    w, ws = codes(40, 8192, 6, dev)
    got = quant8.matmul_8bit(x, xs, w, ws, dtype=BF16)
    for part in (slice(0, 70), slice(FAR - 740, FAR)):
        assert torch.equal(got[part], quant8.matmul_8bit(x[part], xs[part], w, ws, dtype=BF16))
    x, xs, w, ws = *codes(70_000, 48, 7, dev), *codes(40_000, 48, 8, dev)
    got = quant8.matmul_8bit(x, xs, w, ws, dtype=F16)
    assert got.numel() * 2 > 1 << 32
    for part in (slice(0, 70), slice(70_000 - 300, 70_000)):
        assert torch.equal(got[part], quant8.matmul_8bit(x[part], xs[part], w, ws, dtype=F16))


def test_norm_past_4_gb(dev):
    g = torch.Generator(dev).manual_seed(9)
    x = torch.randn((FAR, 8192), dtype=BF16, generator=g, device=dev)
    weight = 1 + 0.3 * torch.randn((8192,), generator=g, device=dev)
    end = slice(FAR - 5, FAR)
    out, few = rows.rms_norm(x, weight, eight_bit=True), rows.rms_norm(x[end], weight, eight_bit=True)
    # (another number of threads a row, sums of squares in another order: results may round to the other side, a step of their type)
    assert torch.equal(out.codes[end], few.codes)
    for a, b, step in ((out.rstd, few.rstd, 2.0 ** -23), (out.scales, few.scales, 2.0 ** -23), (out.y, few.y, 2.0 ** -7)):
        oracle.close(a[end], b.cpu().double(), step * b.cpu().double().abs())
    dy = torch.zeros_like(x)
    dy[end] = torch.randn((5, 8192), dtype=BF16, generator=g, device=dev)
    dx, dw = rows.rms_norm_backward(dy, x, out.rstd, weight)
    assert not bool(dx[:-5].any())
    (want, off), (dw_want, dw_off) = oracle.norm_backward(dy[end], x[end], out.rstd[end], weight, None)
    oracle.close(dx[end], want, off)
    oracle.close(dw, dw_want, dw_off)
