"""What the 4-bit entry points refuse, on the CPU: at the C boundary before any device access, and in the Python layer
before the library is called."""

import pytest
import torch

from scratchtape_amd import _lib, kv4, quant4

FAKE = 1 << 20  # aligned non-null stand-in: every call below is refused before any access


def refused(name, args, message):
    L = _lib.lib()
    assert getattr(L, name)(*args) == _lib.ST_ERR_INVALID, args
    assert message in L.st_last_error().decode(), (args, L.st_last_error())


def swap(args, **kw):
    return [kw.get(k, v) for k, v in args.items()]


def test_quantize_refusals():
    ok = dict(x=FAKE, dtype=0, n=4, k=128, x_stride=128, group=64, codes=FAKE, scales=FAKE, values=None, stream=None)
    for kw, msg in [(dict(group=48), "group"), (dict(group=256), "group"), (dict(k=96), "multiple"), (dict(k=0), "k 0"), (dict(n=-1), "n -1"),
                    (dict(x_stride=127), "apart"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(x=None), "NULL"),
                    (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(x=FAKE + 2), "aligned"),
                    (dict(codes=FAKE + 2), "aligned"), (dict(scales=FAKE + 4), "aligned"), (dict(values=FAKE + 1), "aligned"),
                    (dict(n=1 << 62), "too many")]:
        refused("st_quantize_4bit", swap(ok, **kw), msg)
    assert _lib.lib().st_quantize_4bit(*swap(ok, n=0, x=None, codes=None, scales=None)) == _lib.ST_OK


def test_matvec_refusals():
    ok = dict(x=FAKE, dtype=1, m=2, k=128, x_stride=128, codes=FAKE, scales=FAKE, group=64, n=8, bias=None, relu=0, out=FAKE,
              out_stride=8, stream=None)
    for kw, msg in [(dict(group=0), "group"), (dict(k=32), "multiple"), (dict(m=-1), "m -1"), (dict(n=-5), "n -5"), (dict(x_stride=64), "apart"),
                    (dict(out_stride=7), "apart"), (dict(dtype=7), "dtype"), (dict(x=None), "NULL"), (dict(codes=None), "NULL"),
                    (dict(scales=None), "NULL"), (dict(out=None), "NULL"), (dict(codes=FAKE + 8), "aligned"),
                    (dict(scales=FAKE + 4), "aligned"), (dict(bias=FAKE + 2), "aligned"), (dict(out=FAKE + 1), "aligned"),
                    (dict(k=1 << 21, x_stride=1 << 21), "2^20"), (dict(m=(1 << 19) + 1), "2^19"),
                    (dict(m=1 << 21), "2^20"), (dict(n=(1 << 28) + 1, out_stride=1 << 30), "2^28")]:
        refused("st_matvec_4bit", swap(ok, **kw), msg)
    for kw in (dict(m=0), dict(n=0)):
        assert _lib.lib().st_matvec_4bit(*swap(ok, x=None, out=None, codes=None, scales=None, **kw)) == _lib.ST_OK


APPEND = dict(q=FAKE, k=FAKE, v=FAKE, dtype=0, n=4, hq=8, hkv=2, hd=64, q_stride=512, k_stride=128, v_stride=128, seq=FAKE, pos=FAKE,
              nseq=2, table=FAKE, max_pages=4, pages=9, page=16, inv_freq=FAKE, rot=64, interleaved=0, k_codes=FAKE, k_scales=FAKE,
              v_codes=FAKE, v_scales=FAKE, q_out=2 * FAKE, k_out=None, v_out=None, stream=None)
ATTEND = dict(q=FAKE, dtype=0, n=4, hq=8, hkv=2, hd=64, q_stride=512, q_start=FAKE, kv_len=FAKE, nseq=2, table=FAKE, max_pages=4,
              pages=9, page=16, k_codes=FAKE, k_scales=FAKE, v_codes=FAKE, v_scales=FAKE, scale=0.1, causal=1, window=0, one=0,
              out=2 * FAKE, lse=None, work=FAKE, work_bytes=1 << 40, stream=None)
SHARED = [(dict(hq=7), "multiple"), (dict(hkv=0), "key heads"), (dict(hd=80), "head width"), (dict(hd=48), "head width"),
          (dict(hd=512), "head width"), (dict(page=8), "power of two"), (dict(page=48), "power of two"), (dict(page=2048), "power of two"),
          (dict(n=-1), "-1"), (dict(dtype=3), "dtype"), (dict(nseq=-1), "sequences"), (dict(pages=-1), "sequences"),
          (dict(max_pages=1 << 30), "2^30"), (dict(max_pages=(1 << 26) + 1, page=16), "2^30"), (dict(table=None), "NULL"), (dict(k_codes=None), "NULL"), (dict(v_scales=None), "NULL"),
          (dict(k_scales=FAKE + 8), "aligned"), (dict(v_codes=FAKE + 4), "aligned"), (dict(q_stride=511), "apart")]


@pytest.mark.parametrize("kw,msg", SHARED + [
    (dict(rot=63), "rotated"), (dict(rot=66), "rotated"), (dict(rot=-2), "rotated"), (dict(inv_freq=None), "NULL"),
    (dict(k_stride=127), "apart"), (dict(v_stride=0), "apart"), (dict(k=None), "NULL"), (dict(v=None), "NULL"),
    (dict(seq=None), "NULL"), (dict(pos=None), "NULL"), (dict(q_out=None), "NULL"), (dict(q_out=FAKE), "memory"),
    (dict(k=FAKE + 2), "aligned"), (dict(q_out=2 * FAKE + 2), "aligned")])
def test_append_refusals(kw, msg):
    refused("st_kv_append_4bit", swap(APPEND, **kw), msg)


@pytest.mark.parametrize("kw,msg", SHARED + [
    (dict(window=-1), "window"), (dict(window=4, causal=0), "window"), (dict(q=None), "NULL"), (dict(out=None), "NULL"),
    (dict(q_start=None), "NULL"), (dict(kv_len=None), "NULL"), (dict(out=2 * FAKE + 1), "aligned"), (dict(q=FAKE + 2), "aligned")])
def test_attention_refusals(kw, msg):
    refused("st_kv_attention_4bit", swap(ATTEND, **kw), msg)


def test_attention_takes_2_to_the_26_rows_of_heads():
    """One more row is refused by its number; as many as that only by what comes after."""
    refused("st_kv_attention_4bit", swap(ATTEND, n=(1 << 23) + 1), "2^26")
    refused("st_kv_attention_4bit", swap(ATTEND, n=1 << 62), "2^26")
    refused("st_kv_attention_4bit", swap(ATTEND, n=1 << 23, out=None), "NULL")


def test_nothing_to_do_is_no_error():
    L = _lib.lib()
    assert L.st_kv_append_4bit(*swap(APPEND, n=0, q=None, k=None, v=None)) == _lib.ST_OK
    assert L.st_kv_attention_4bit(*swap(ATTEND, n=0, q=None, out=None)) == _lib.ST_OK


def test_python_refuses_before_the_library(monkeypatch):
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("reached the library"))
    x = torch.zeros(4, 128)
    for bad, msg in [((x.double(),), "float32"), ((x[0],), "n, k"), ((x, 48), "group"), ((x[:, :96], 64), "multiple"), ((x.t(), 32), "multiple|contiguous"),
                     ((x[:, ::2], 64), "contiguous"), ((x, 64, x), "shares memory"), ((x, 64, x.half()), "values"), ((x,), "GPU")]:
        with pytest.raises(ValueError, match=msg):
            quant4.quantize_4bit(*bad)
    with pytest.raises(ValueError, match="overlap"):
        quant4.quantize_4bit(torch.zeros(400).as_strided((4, 128), (64, 1)))
    codes, scales = torch.zeros(6, 64, dtype=torch.uint8), torch.zeros(6, 2, 2)
    for bad, msg in [((x[:, :64], codes, scales), "codes"), ((x, codes.int(), scales), "codes"), ((x, codes, scales[:5]), "scales"),
                     ((x, codes, torch.zeros(6, 3, 2)), "scales"), ((x, codes, torch.zeros(6, 8, 2)), "groups of 16"),
                     ((x, codes, scales, torch.zeros(5)), "bias"), ((x, codes, scales, None, False, torch.zeros(4, 5)), "out is"),
                     ((x, codes, scales, None, False, torch.zeros(4, 6).half()), "out is"),
                     ((x, codes, scales, None, False, x[:, :6]), "shares memory"), ((x, codes, scales), "GPU")]:
        with pytest.raises(ValueError, match=msg):
            quant4.matvec_4bit(*bad)


def test_cache_refusals(monkeypatch):
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("reached the library"))
    for pages, heads, page, hd, msg in [(3, 2, 24, 64, "power of two"), (3, 2, 8, 64, "power of two"), (3, 2, 16, 80, "head width"),
                                        (3, 0, 16, 64, "one head")]:
        with pytest.raises(ValueError, match=msg):
            kv4.KvCache4bit.empty(pages, heads, page, hd, "cpu")
    cache = kv4.KvCache4bit.empty(3, 2, 16, 64, "cpu")
    with pytest.raises(ValueError, match="v_scales"):
        kv4.KvCache4bit(cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales[:2])
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    q, k, table = torch.zeros(4, 6, 64), torch.zeros(4, 2, 64), torch.zeros(2, 2, dtype=torch.int32)
    seq = i(0, 0, 1, 1)
    ok = dict(q=q, k=k, v=k.clone(), seq=seq, pos=seq, table=table, inv_freq=torch.zeros(32))
    for kw, msg in [(dict(k=torch.zeros(4, 3, 64)), "k is"), (dict(q=torch.zeros(4, 5, 64)), "q is"), (dict(q=torch.zeros(3, 6, 64)), "q is"),
                    (dict(v=k.half()), "same type"), (dict(v=torch.zeros(5, 2, 64)), "same tokens"), (dict(seq=seq.long()), "seq"),
                    (dict(pos=seq[:3]), "pos"), (dict(table=table.long()), "table"), (dict(table=table[0]), "table"),
                    (dict(inv_freq=torch.zeros(33)), "rotates"), (dict(inv_freq=torch.zeros(32).double()), "inv_freq"),
                    (dict(out=[q]), "shares memory"), (dict(out=[k]), "out"), (dict(out=[None, k]), "out holds"),
                    (dict(values=True, out=[None, torch.zeros(4, 2, 64).half()]), "out"), (dict(q=None, out=[q]), "without q"),
                    (dict(k=torch.zeros(4, 64, 2).transpose(1, 2)), "contiguous"), ({}, "GPU")]:
        with pytest.raises(ValueError, match=msg):
            cache.append(**{**ok, **kw})
    ok = dict(q=q, table=table, q_start=i(0, 2, 4), kv_len=i(5, 5))
    for kw, msg in [(dict(q=torch.zeros(4, 5, 64)), "multiple"), (dict(q=torch.zeros(4, 6, 32)), "q is"), (dict(q_start=i(0, 4)), "q_start"),
                    (dict(kv_len=i(5)), "kv_len"), (dict(kv_len=torch.zeros(2)), "kv_len"), (dict(window=-1), "window"),
                    (dict(window=3, causal=False), "window"), (dict(out=q), "shares memory"), (dict(out=torch.zeros(4, 6, 64).half()), "out"),
                    (dict(q=q.double()), "float32"), ({}, "GPU")]:
        with pytest.raises(ValueError, match=msg):
            cache.attention(**{**ok, **kw})
