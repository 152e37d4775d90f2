"""Which kernel an 8-bit product takes, asked on the host: every kernel is some shape's, slices leave stages to each, and the
work memory follows the plan."""
import itertools
import os
import subprocess

import pytest

from scratchtape_amd import _lib, build, quant8
import test_lds_waits

SIZES = [(m, k, n) for m, k, n in itertools.product((1, 2, 4, 5, 16, 17, 33, 64, 65, 200, 512, 1024, 4096, 8192), (16, 100, 512, 1000, 4096, 16384, 131072),
                                                    (1, 16, 300, 1024, 8192, 30000))]


@pytest.mark.parametrize("gated", [False, True])
def test_every_kernel_is_taken(gated):
    plans = {s: quant8.product_plan(*s, gated=gated) for s in SIZES}
    kernels = {kernel for kernel, _ in plans.values()}
    # 64 x 64 tiles do a gated product by slices alone: a wave of theirs does not hold both halves
    assert kernels == ({"one", "few", "large", "middle", "low", "deep_low", "small", "deep"} if gated else
                       {"one", "few", "large", "middle", "small", "deep"})
    for (m, k, n), (kernel, slices) in plans.items():
        assert kernel != "one" or m <= 4
        assert kernel != "few" or m <= 32
        assert (kernel in ("deep", "deep_low")) <= (m <= 64) and (kernel in ("small", "middle", "large", "low")) <= (m > 64)
        assert slices == 1 or kernel in ("small", "deep")
        if gated and kernel in ("small", "deep"):
            assert slices > 1
        assert 1 <= slices <= 16 and slices <= max(1, k // 256)
        need = _lib.lib().st_matmul_8bit_bytes(m, k, n, int(gated))
        assert need == (0 if slices == 1 else 4 * slices * m * n * (2 if gated else 1))


def test_plan_refusals():
    for bad in ((0, 5, 5), (5, 0, 5), (5, 5, 0), (5, 131073, 5), (-1, 5, 5), ((1 << 30) + 1, 5, 5), (5, 5, (1 << 30) + 1)):
        with pytest.raises(_lib.ScratchtapeError, match="matmul_8bit_plan"):
            quant8.product_plan(*bad)
        assert _lib.lib().st_matmul_8bit_bytes(*bad, 0) == 0
    assert _lib.lib().st_matmul_8bit_bytes(1 << 40, 64, 1 << 40, 0) == 0


def test_launches_stay_within_2_to_the_32_threads():
    """The kernel for few rows has a workgroup of up to 512 threads for 16 rows of weights, and is not taken where that is too many."""
    for n in (1 << 27, (1 << 30) - 5):
        for m in (1, 7, 32):
            for gated in (False, True):
                assert quant8.product_plan(m, 16, n, gated)[0] != "few"


@pytest.mark.skipif(test_lds_waits.HIPCC is None, reason="needs hipcc")
def test_no_lds_write_is_in_flight_at_a_barrier(tmp_path):
    """The tiles' kernels have barriers without __syncthreads' fence: no LDS write of a wave is in flight at one."""
    out = str(tmp_path / "k.s")
    flags = [f for f in build.CFLAGS if f != "-fPIC"]
    subprocess.run([test_lds_waits.HIPCC, *flags, "-S", "--cuda-device-only", os.path.join(build.CSRC, "matmul8.hip"), "-o", out], check=True,
                   capture_output=True)
    found = {n: l for n, l in test_lds_waits.kernels(open(out).read()).items() if "s_barrier" in l}
    assert len(found) >= 20, list(found)
    bad = {n: b for n, l in found.items() if (b := test_lds_waits.barriers_with_writes_in_flight(l))}
    assert not bad, f"{len(bad)} of {len(found)} kernels: {bad}"
