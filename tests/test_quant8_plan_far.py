"""What an 8-bit product's plan answers where a tile's 32-bit offsets end: the kernel for any strides, which is what runs."""
import pytest
import torch

from scratchtape_amd import _lib, quant8

TILES = {"large", "middle", "low", "small", "deep", "deep_low"}
WIDE = 1 << 21  # columns of a contiguous out
HALF = (2 ** 32 - 2 ** 16) // 8192 - 256  # gated columns of 8192 codes each whose two halves are too far apart


@pytest.mark.parametrize("m,k,n,gated", [(64, 64, WIDE, False), (40, 48, WIDE + 5, False), (200, 16, WIDE, False), (65, 100, WIDE, True), (33, 64, 2 * WIDE, True),
                                         (70, 8192, HALF, True), (5000, 8190, HALF + 1, True), (40, 8192, HALF, True)])
def test_far_products_take_the_kernel_for_any_strides(m, k, n, gated):
    assert quant8.product_plan(m, k, n, gated) == ("any", 1)
    assert _lib.lib().st_matmul_8bit_bytes(m, k, n, int(gated)) == 0
    edge = (WIDE if n >= WIDE else HALF) - 1
    assert quant8.product_plan(m, k, edge, gated)[0] in TILES


def test_kernels_without_tiles_go_on():
    assert quant8.product_plan(1, 8192, 2 * WIDE)[0] == quant8.product_plan(4, 8192, HALF, True)[0] == "one"
    assert {quant8.product_plan(*s)[0] for s in ((8, 64, 2 * WIDE), (32, 4096, WIDE), (16, 8192, HALF, True), (32, 8192, HALF, True))} == {"few"}


@pytest.mark.gpu
def test_wide_outputs(dev):
    g = torch.Generator(dev).manual_seed(1)
    for m in (40, 20):
        wide_output(g, m, 48, WIDE + 5, dev)


def wide_output(g, m, k, n, dev):
    x, w = (torch.randint(-127, 128, (rows, k), generator=g, device=dev, dtype=torch.int8) for rows in (m, n))
    xs, ws = (torch.rand(rows, generator=g, device=dev) for rows in (m, n))
    got = quant8.matmul_8bit(x, xs, w, ws, dtype=torch.float32)
    for part in (slice(0, 70), slice(n - 700, n)):
        assert torch.equal(got[:, part], quant8.matmul_8bit(x, xs, w[part], ws[part], dtype=torch.float32))
