"""A paged cache of keys and values in 4 bits on MI355X, and attention over it: one layer's side of running a model token
by token (no reference counterpart; the training side is attention.py).

The cache holds [pages, heads, page, ...] codes and scales; a token's head vector is one group of the 4-bit format of
quant4.py.  Token p of sequence s is in page table[s, p // page], slot p % page.  A decoding step appends its tokens
(queries and keys rotated by their positions) and attends; both read sequences, positions, lengths and pages on the
device, so a captured graph follows them.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _lib
from .quant4 import _addr, _apart, _dtype, _launch, _on_gpu, _plain, _rows

HEAD_DIMS = (32, 64, 96, 128, 192, 256)


@dataclass
class KvCache4bit:
    """One layer's cache: codes [pages, heads, page, hd/2] uint8 and scales [pages, heads, page, 2] float32 (scale, lo) of
    the keys and of the values.  hd is one of HEAD_DIMS, page a power of two from 16 to 1024 tokens."""
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor

    def __post_init__(self):
        if not isinstance(self.k_codes, torch.Tensor) or self.k_codes.dim() != 4:
            raise ValueError("k_codes is [pages, heads, page, hd / 2]")
        pages, heads, page, half = self.k_codes.shape
        for t, name in ((self.k_codes, "k_codes"), (self.v_codes, "v_codes")):
            _plain(t, torch.uint8, (pages, heads, page, half), name)
        for t, name in ((self.k_scales, "k_scales"), (self.v_scales, "v_scales")):
            _plain(t, torch.float32, (pages, heads, page, 2), name)
        if 2 * half not in HEAD_DIMS:
            raise ValueError(f"head width {2 * half} is none of {HEAD_DIMS}")
        if page < 16 or page > 1024 or page & (page - 1):
            raise ValueError(f"pages of {page} tokens: a power of two from 16 to 1024 is taken")
        if heads < 1:
            raise ValueError("a cache has one head at least")

    @staticmethod
    def empty(pages: int, heads: int, page: int, hd: int, device) -> "KvCache4bit":
        z = lambda *shape, **kw: torch.zeros(shape, device=device, **kw)
        codes = lambda: z(pages, heads, page, hd // 2, dtype=torch.uint8)
        return KvCache4bit(codes(), z(pages, heads, page, 2), codes(), z(pages, heads, page, 2))

    def _buffers(self):
        return [(self.k_codes, "k_codes"), (self.k_scales, "k_scales"), (self.v_codes, "v_codes"), (self.v_scales, "v_scales")]

    def _heads(self, t: torch.Tensor, heads: Optional[int], what: str):
        """(tokens, heads, row stride) of a [n, heads, hd] tensor."""
        hd = 2 * self.k_codes.shape[3]
        if t.dim() != 3 or t.shape[2] != hd or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"{what} is [tokens, {'heads' if heads is None else heads}, {hd}], got {list(t.shape)}")
        return t.shape[0], t.shape[1], _rows(t, what)

    def _table(self, table: torch.Tensor):
        if not isinstance(table, torch.Tensor) or table.dim() != 2:
            raise ValueError("table is [sequences, pages of a sequence]")
        return _plain(table, torch.int32, table.shape, "table").shape

    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor,
               table: torch.Tensor, inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False, values: bool = False,
               out: Optional[Sequence[Optional[torch.Tensor]]] = None, stream=None):
        """Appends tokens: token t is at position pos[t] of sequence seq[t] (both int32 [n]), its queries q [n, hq, hd] and
        keys k [n, heads, hd] rotated by pos[t] * inv_freq[i] (float32 [rot / 2], rot <= hd; None: not rotated), component
        pairs (i, i + rot / 2), or (2i, 2i + 1) where interleaved; keys and values v are quantised into the cache.  Tokens
        may be any number of elements apart (views of a fused projection).

        Returns the rotated queries (None without q), and with `values` a list of them, the keys and the values as the cache
        now holds them, in the inputs' type.  out: tensors to fill, in that order.  A token of no sequence (seq outside
        the table, such as -1 for padding), at no place of the table or on a page outside the cache writes nothing (its rows
        of new tensors hold whatever their memory held); no two tokens of a call may name the same place."""
        pages, heads, page, half = self.k_codes.shape
        dtype = _dtype(k, "k")
        n, _, k_stride = self._heads(k, heads, "k")
        nv, _, v_stride = self._heads(v, heads, "v")
        hq, q_stride = heads, 0
        if q is not None:
            nq, hq, q_stride = self._heads(q, None, "q")
            if nq != n or hq < 1 or hq % heads:
                raise ValueError(f"q is [{n}, a multiple of {heads}, {2 * half}], got {list(q.shape)}")
        if nv != n or _dtype(v, "v") != dtype or (q is not None and _dtype(q, "q") != dtype):
            raise ValueError("q, k and v hold the same tokens in the same type")
        for t, name in ((seq, "seq"), (pos, "pos")):
            _plain(t, torch.int32, (n,), name)
        nseq, max_pages = self._table(table)
        rot = 0
        if inv_freq is not None:
            rot = 2 * inv_freq.numel()
            _plain(inv_freq, torch.float32, (rot // 2,), "inv_freq")
            if rot > 2 * half:
                raise ValueError(f"inv_freq rotates {rot} components of {2 * half}")
        shapes = [None if q is None else (n, hq, 2 * half), (n, heads, 2 * half), (n, heads, 2 * half)]
        outs = list(out) if out is not None else []
        if len(outs) > (3 if values else 1):
            raise ValueError("out holds the rotated queries, and with values the keys and the values")
        outs += [None] * (3 - len(outs))
        for t, shape, name in zip(outs, shapes, ("out[0]", "out[1]", "out[2]")):
            if t is not None:
                if shape is None:
                    raise ValueError("out[0] is given without q")
                _plain(t, k.dtype, shape, name)
        ins = [(q, "q"), (k, "k"), (v, "v"), (seq, "seq"), (pos, "pos"), (table, "table"), (inv_freq, "inv_freq")]
        written = [(outs[0], "out[0]"), (outs[1], "out[1]"), (outs[2], "out[2]")] + self._buffers()
        _apart(written, ins)
        _on_gpu(k, ins + written)
        with _launch(k.device, stream) as handle:
            wanted = (True, values, values)
            q_out, k_out, v_out = (t if t is not None or shape is None or not want else
                                   torch.empty(shape, dtype=k.dtype, device=k.device)
                                   for t, shape, want in zip(outs, shapes, wanted))
            _lib.call("st_kv_append_4bit", _addr(q), k.data_ptr(), v.data_ptr(), dtype, n, hq, heads, 2 * half, q_stride,
                      k_stride, v_stride, seq.data_ptr(), pos.data_ptr(), nseq, table.data_ptr(), max_pages, pages, page,
                      _addr(inv_freq), rot, int(bool(interleaved)), self.k_codes.data_ptr(), self.k_scales.data_ptr(),
                      self.v_codes.data_ptr(), self.v_scales.data_ptr(), _addr(q_out), _addr(k_out), _addr(v_out), handle)
        return [q_out, k_out, v_out] if values else q_out

    def attention(self, q: torch.Tensor, table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
                  scale: Optional[float] = None, causal: bool = True, window: int = 0, one: bool = False, lse: bool = False,
                  out: Optional[torch.Tensor] = None, stream=None):
        """softmax(scale q k^T) v for rows q [n, hq, hd] (rotated): sequence s has the rows q_start[s] .. q_start[s + 1]
        (int32 [sequences + 1]) and kv_len[s] (int32) cached tokens, its own rows' the last of them (n * hq up to 2^26).  A row sees the tokens
        up to its own position (causal; else all), the last `window` of those if window > 0.  scale: hd ** -0.5 unless
        given; one: softmax1.  Returns [n, hq, hd] in q's type (`out` if given), with lse also the log-sum-exp of the
        scores, float32 [n, hq].  A row that sees no token gets 0 and -inf (0 with softmax1); one that sees a token on a
        page outside the cache, or past its table, NaN.  Rows that no sequence has are left as they were (in new
        tensors: whatever their memory held)."""
        pages, heads, page, half = self.k_codes.shape
        dtype = _dtype(q, "q")
        n, hq, q_stride = self._heads(q, None, "q")
        if hq < 1 or hq % heads:
            raise ValueError(f"{hq} query heads over {heads} key heads: a multiple is taken")
        nseq, max_pages = self._table(table)
        _plain(q_start, torch.int32, (nseq + 1,), "q_start")
        _plain(kv_len, torch.int32, (nseq,), "kv_len")
        if window < 0 or (window > 0 and not causal):
            raise ValueError(f"a window of {window} keys goes with the causal mask")
        ins = [(q, "q"), (table, "table"), (q_start, "q_start"), (kv_len, "kv_len")] + self._buffers()
        if out is not None:
            _plain(out, q.dtype, (n, hq, 2 * half), "out")
            _apart([(out, "out")], ins)
        _on_gpu(q, ins + [(out, "out")])
        with _launch(q.device, stream) as handle:
            if out is None:
                out = torch.empty((n, hq, 2 * half), dtype=q.dtype, device=q.device)
            stats = torch.empty((n, hq), dtype=torch.float32, device=q.device) if lse else None
            nbytes = int(_lib.lib().st_kv_attention_4bit_bytes(dtype, n, nseq, hq, heads, 2 * half, max_pages, page))
            work = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes > 0 else None
            _lib.call("st_kv_attention_4bit", q.data_ptr(), dtype, n, hq, heads, 2 * half, q_stride, q_start.data_ptr(),
                      kv_len.data_ptr(), nseq, table.data_ptr(), max_pages, pages, page,
                      self.k_codes.data_ptr(), self.k_scales.data_ptr(), self.v_codes.data_ptr(), self.v_scales.data_ptr(), float((2 * half) ** -0.5 if scale is None else scale),
                      int(bool(causal)), int(window), int(bool(one)), out.data_ptr(), _addr(stats), _addr(work), nbytes,
                      handle)
        return (out, stats) if lse else out
