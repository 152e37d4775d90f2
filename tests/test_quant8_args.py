"""What the 8-bit entry points and the norm's refuse, on the CPU: at the C boundary before any device access, and in the
Python layer before the library is called."""

import pytest
import torch

from scratchtape_amd import _lib, quant8, rows

FAKE = 1 << 20  # aligned non-null stand-in: every call below is refused before any access


def refused(name, args, message):
    L = _lib.lib()
    assert getattr(L, name)(*args) == _lib.ST_ERR_INVALID, args
    assert message in L.st_last_error().decode(), (args, L.st_last_error())


def swap(args, **kw):
    assert not set(kw) - set(args)
    return [kw.get(k, v) for k, v in args.items()]


def test_quantize_refusals():
    ok = dict(x=FAKE, dtype=0, n=4, k=100, x_stride=100, codes=FAKE, codes_stride=112, scales=FAKE, values=None, stream=None)
    for kw, msg in [(dict(k=0), "k 0"), (dict(n=-1), "n -1"), (dict(n=1 << 62), "2^36"), (dict(k=1 << 31), "2^30"), (dict(x_stride=99), "apart"),
                    (dict(codes_stride=99), "apart"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(x=None), "NULL"),
                    (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(x=FAKE + 2), "aligned"), (dict(values=FAKE + 2), "aligned"),
                    (dict(dtype=1, x=FAKE + 1), "aligned"), (dict(scales=FAKE + 2), "aligned")]:
        refused("st_quantize_8bit", swap(ok, **kw), msg)
    assert _lib.lib().st_quantize_8bit(*swap(ok, n=0, x=None, codes=None, scales=None)) == _lib.ST_OK


def test_norm_refusals():
    ok = dict(x=FAKE, residual=FAKE, dtype=1, rows=4, d=100, x_stride=100, residual_stride=100, weight=FAKE, weight_dtype=1, eps=1e-5, h=FAKE,
              rstd=FAKE, y=FAKE, codes=FAKE, codes_stride=100, scales=FAKE, values=FAKE, stream=None)
    for kw, msg in [(dict(d=0), "d 0"), (dict(rows=-1), "rows -1"), (dict(rows=1 << 40), "2^36"), (dict(d=1 << 31, x_stride=1 << 31), "2^30"),
                    (dict(x_stride=99), "apart"), (dict(residual_stride=99), "apart"), (dict(codes_stride=99), "apart"), (dict(dtype=3), "dtype"),
                    (dict(weight_dtype=2), "weight"), (dict(weight_dtype=5), "weight"), (dict(eps=-1e-5), "eps"), (dict(eps=float("nan")), "eps"),
                    (dict(eps=float("inf")), "eps"), (dict(x=None), "NULL"), (dict(weight=None), "NULL"), (dict(scales=None), "NULL"),
                    (dict(codes=None), "NULL"), (dict(codes=None, scales=None), "values"),
                    (dict(codes=None, scales=None, values=None, h=None, y=None, rstd=None), "no output"), (dict(x=FAKE + 1), "aligned"),
                    (dict(residual=FAKE + 1), "aligned"), (dict(weight=FAKE + 1), "aligned"), (dict(weight_dtype=0, weight=FAKE + 2), "aligned"),
                    (dict(h=FAKE + 1), "aligned"), (dict(y=FAKE + 1), "aligned"), (dict(values=FAKE + 1), "aligned"), (dict(rstd=FAKE + 2), "aligned"),
                    (dict(scales=FAKE + 2), "aligned")]:
        refused("st_rms_norm", swap(ok, **kw), msg)
    assert _lib.lib().st_rms_norm(*swap(ok, rows=0, x=None, weight=None)) == _lib.ST_OK


def test_backward_refusals():
    ok = dict(dy=FAKE, h=FAKE, dh=FAKE, dtype=0, rows=5000, d=64, dy_stride=64, h_stride=64, dh_stride=64, rstd=FAKE, weight=FAKE, weight_dtype=0,
              dx=FAKE, dweight=FAKE, work=FAKE, work_bytes=1 << 40, stream=None)
    assert _lib.lib().st_rms_norm_backward_bytes(5000, 64, 0) > 0
    assert [_lib.lib().st_rms_norm_backward_bytes(*v, 1) for v in ((1, 64), (0, 64), (-1, 64), (5, 0), (1 << 40, 64))] == 5 * [0]
    for kw, msg in [(dict(d=0), "d 0"), (dict(rows=-1), "rows -1"), (dict(dy_stride=63), "apart"), (dict(h_stride=63), "apart"), (dict(dh_stride=63), "apart"),
                    (dict(dtype=3), "dtype"), (dict(dtype=1, weight_dtype=2), "weight"), (dict(dy=None), "NULL"), (dict(h=None), "NULL"),
                    (dict(rstd=None), "NULL"), (dict(weight=None), "NULL"), (dict(dx=None), "NULL"), (dict(dweight=None), "NULL"),
                    (dict(work=None), "work memory"), (dict(work_bytes=100), "work memory"), (dict(work=FAKE + 8), "aligned"),
                    (dict(dx=FAKE + 2), "aligned"), (dict(dy=FAKE + 2), "aligned"), (dict(dh=FAKE + 2), "aligned"), (dict(dweight=FAKE + 2), "aligned")]:
        refused("st_rms_norm_backward", swap(ok, **kw), msg)


PRODUCT = dict(x=FAKE, x_scales=FAKE, m=4, k=100, x_stride=112, w=FAKE, w_scales=FAKE, n=8, w_stride=112, bias=None, act=0, out=FAKE, dtype=1,
               out_stride=8, work=FAKE, work_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("name,act", [("st_matmul_8bit", 0), ("st_gated_8bit", 2)])
def test_product_refusals(name, act):
    ok = dict(PRODUCT, act=act)
    for kw, msg in [(dict(m=-1), "m -1"), (dict(n=-5), "n -5"), (dict(k=0), "k 0"), (dict(k=131073, x_stride=1 << 20, w_stride=1 << 20), "131072"),
                    (dict(m=1 << 31), "too many"), (dict(m=1 << 20, n=1 << 20, out_stride=1 << 20), "too many"), (dict(x_stride=99), "apart"), (dict(w_stride=99), "apart"),
                    (dict(out_stride=7), "apart"), (dict(dtype=3), "dtype"), (dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(x_scales=None), "NULL"),
                    (dict(w_scales=None), "NULL"), (dict(out=None), "NULL"), (dict(out=FAKE + 1), "aligned"), (dict(bias=FAKE + 2), "aligned"),
                    (dict(x_scales=FAKE + 2), "aligned"), (dict(w_scales=FAKE + 1), "aligned"), (dict(work=FAKE + 4), "aligned")]:
        refused(name, swap(ok, **kw), msg)
    for kw in (dict(m=0), dict(n=0)):
        assert getattr(_lib.lib(), name)(*swap(ok, x=None, w=None, out=None, **kw)) == _lib.ST_OK


def test_gated_takes_its_own_activations():
    for act in (0, 1, 4, -1):
        refused("st_gated_8bit", swap(PRODUCT, act=act), "activation")


def test_python_refuses_before_the_library(monkeypatch):
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("reached the library"))
    x = torch.zeros(4, 128)
    for bad, msg in [((x.double(),), "float32"), ((x[0],), "n, k"), ((x[:, :0],), "n, k"), ((x.t(),), "contiguous"), ((x[:, ::2],), "contiguous"),
                     ((x, x), "shares memory"), ((x, x.half()), "values"), ((x, x[:3].clone()), "values"), ((x,), "GPU")]:
        with pytest.raises(ValueError, match=msg):
            quant8.quantize_8bit(*bad)
    with pytest.raises(TypeError):
        quant8.quantize_8bit([1.0])
    c, w, s, ws = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(6, 64, dtype=torch.int8), torch.zeros(4), torch.zeros(6)
    ok = dict(x=c, x_scales=s, w=w, w_scales=ws)
    for kw, msg in [(dict(x=c.int()), "int8"), (dict(w=w.to(torch.uint8)), "int8"), (dict(x=c[0]), "int8"), (dict(w=w[:, :32]), "columns"),
                    (dict(x_scales=ws), "x_scales"), (dict(w_scales=s), "w_scales"), (dict(x_scales=s.half()), "x_scales"), (dict(bias=s), "bias"),
                    (dict(dtype=torch.float64), "dtype"), (dict(dtype=torch.int8), "dtype"), (dict(out=torch.zeros(4, 6)), "out is"),
                    (dict(x=torch.zeros(64, 4, dtype=torch.int8).t()), "contiguous"), ({}, "GPU")]:
        for call in (quant8.matmul_8bit, quant8.gated_8bit):
            with pytest.raises(ValueError, match=msg):
                call(**{**ok, **kw})
    with pytest.raises(ValueError, match="out is"):
        quant8.matmul_8bit(**ok, dtype=torch.float32, out=torch.zeros(4, 5))
    with pytest.raises(ValueError, match="shares memory"):
        quant8.matmul_8bit(**ok, dtype=torch.float32, out=_over(w))
    with pytest.raises(ValueError, match="activation"):
        quant8.gated_8bit(**ok, activation="relu")
    with pytest.raises(ValueError, match="as many more"):
        quant8.gated_8bit(**{**ok, "w": w[:5], "w_scales": ws[:5]})
    with pytest.raises(TypeError):
        quant8.matmul_8bit(c, s, None, ws)


def _over(w):
    """Outputs [4, 6] float32 in the memory of the weights."""
    return w.view(torch.float32).flatten()[:24].view(4, 6)


def test_python_norm_refusals(monkeypatch):
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("reached the library"))
    x, w = torch.zeros(4, 96).half(), torch.ones(96)
    for kw, msg in [(dict(x=x.double()), "float32"), (dict(x=x[0]), "rows, d"), (dict(x=x[:, :0]), "rows, d"), (dict(weight=w[:95]), "weight"),
                    (dict(weight=w.bfloat16()), "weight"), (dict(weight=w.double()), "weight"), (dict(residual=x[:3]), "residual"),
                    (dict(residual=x.float()), "residual"), (dict(eps=-1.0), "eps"), (dict(values=True), "eight_bit"), (dict(y=False), "neither"), (dict(x=x.t()), "weight|contiguous"),
                    ({}, "GPU")]:
        with pytest.raises(ValueError, match=msg):
            rows.rms_norm(**{**dict(x=x, weight=w), **kw})
    ok = dict(dy=x, h=x, rstd=torch.zeros(4), weight=w)
    for kw, msg in [(dict(dy=x.float()), "dy"), (dict(dy=x[:2]), "dy"), (dict(rstd=torch.zeros(5)), "rstd"), (dict(dh=x[:, :5]), "dh"),
                    (dict(weight=w[:4]), "weight"), (dict(h=x[0]), "rows, d"), ({}, "GPU")]:
        with pytest.raises(ValueError, match=msg):
            rows.rms_norm_backward(**{**ok, **kw})
    with pytest.raises(TypeError):
        rows.rms_norm(x, None)
    with pytest.raises(TypeError):
        rows.rms_norm_backward(None, x, torch.zeros(4), w)
