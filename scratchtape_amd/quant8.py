"""8-bit rows on MI355X: the quantiser of weights and activations, and Linear layers of 8-bit weights on 8-bit rows, from one
token to long prompts (no reference counterpart; `rows.rms_norm` makes 8-bit rows of normed activations).

A row x has a = max |x| and scale = f32(a / 127); a value is held as code = round_half_even(127 x / a), decided in 64 bits,
and stands for scale * code.  Codes are int8 [rows, k], scales float32 [rows].  A row that holds a NaN or an infinity has
scale NaN and codes 0, so that what is computed from it is NaN.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .quant4 import DTYPES, _addr, _apart, _dtype, _launch, _on_gpu, _plain, _rows

ACTIVATIONS = {"silu": 2, "gelu": 3}  # ST_ACT_SILU, ST_ACT_GELU


def empty_codes(rows: int, k: int, device) -> torch.Tensor:
    """Room for codes [rows, k] whose rows are 16-byte aligned, as the products read them fastest."""
    return torch.empty((rows, (k + 15) // 16 * 16), dtype=torch.int8, device=device)[:, :k]


def _new_codes(rows: int, k: int, like: torch.Tensor) -> torch.Tensor:
    """empty_codes where `like` is."""
    width = (k + 15) // 16 * 16
    codes = like.new_empty((rows, width), dtype=torch.int8)
    return codes if width == k else codes[:, :k]


def quantize_8bit(x: torch.Tensor, values: Union[bool, torch.Tensor] = False, stream=None):
    """Rows x [n, k] (any row stride) -> codes [n, k] int8 and scales [n] float32.

    values: also return what the codes stand for, [n, k] in x's type (True: a new tensor, or a tensor to fill), the
    forward value of a straight-through gradient.  Rows of codes are a multiple of 16 bytes apart."""
    dtype = _dtype(x, "x")
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"x is [n, k] with k > 0, got {list(x.shape)}")
    n, k = x.shape
    stride = _rows(x, "x")
    out = values if isinstance(values, torch.Tensor) else None
    if out is not None:
        _plain(out, x.dtype, (n, k), "values")
        _apart([(out, "values")], [(x, "x")])
    _on_gpu(x, [(out, "values")])
    with _launch(x.device, stream) as handle:
        codes, scales = _new_codes(n, k, x), x.new_empty((n,), dtype=torch.float32)
        if out is None and values:
            out = x.new_empty((n, k))
        _lib.call("st_quantize_8bit", x.data_ptr(), dtype, n, k, stride, codes.data_ptr(), (k + 15) // 16 * 16, scales.data_ptr(),
                  _addr(out), handle)
    return (codes, scales) if out is None else (codes, scales, out)


def _codes(t: torch.Tensor, what: str) -> Tuple[int, int, int]:
    """Rows, width and row stride of a tensor of codes."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} is a torch tensor")
    if t.dtype != torch.int8 or t.dim() != 2 or t.shape[1] == 0:
        raise ValueError(f"{what} is int8 [rows, k] with k > 0; got {t.dtype} {list(t.shape)}")
    return t.shape[0], t.shape[1], _rows(t, what)


def _product(name, x, x_scales, w, w_scales, bias, flag, halves, dtype, out, stream):
    m, k, x_stride = _codes(x, "x")
    width, wk, w_stride = _codes(w, "w")
    if wk != k:
        raise ValueError(f"x has {k} columns, w {wk}")
    if width % halves:
        raise ValueError(f"w holds the gate's rows and as many more; got {width} rows")
    n = width // halves
    _plain(x_scales, torch.float32, (m,), "x_scales")
    _plain(w_scales, torch.float32, (width,), "w_scales")
    if bias is not None:
        _plain(bias, torch.float32, (width,), "bias")
    if out is None:
        if dtype not in DTYPES:
            raise ValueError(f"dtype is {dtype}; float32, float16 and bfloat16 are taken")
    else:
        if _dtype(out, "out") != DTYPES.get(dtype) or tuple(out.shape) != (m, n):
            raise ValueError(f"out is {dtype} [{m}, {n}]; got {out.dtype} {list(out.shape)}")
        out_stride = _rows(out, "out")
        _apart([(out, "out")], [(x, "x"), (x_scales, "x_scales"), (w, "w"), (w_scales, "w_scales"), (bias, "bias")])
    _on_gpu(x, [(x_scales, "x_scales"), (w, "w"), (w_scales, "w_scales"), (bias, "bias"), (out, "out")])
    with _launch(x.device, stream) as handle:
        if out is None:
            out, out_stride = x_scales.new_empty((m, n), dtype=dtype), n
        need = _lib.lib().st_matmul_8bit_bytes(m, k, n, halves - 1)
        work = x.new_empty((need,)) if need else None
        _lib.call(name, x.data_ptr(), x_scales.data_ptr(), m, k, x_stride, w.data_ptr(), w_scales.data_ptr(), n, w_stride, _addr(bias), flag,
                  out.data_ptr(), DTYPES[dtype], out_stride, _addr(work), need, handle)
    return out


KERNELS = ("one", "few", "large", "middle", "low", "small", "deep", "deep_low", "any")


def product_plan(m: int, k: int, n: int, gated: bool = False) -> Tuple[str, int]:
    """The kernel (of KERNELS) that matmul_8bit, or gated_8bit, takes for x [m, k] and n columns of out where codes lie as
    quantize_8bit lays them and out is contiguous, and into how many slices it cuts k.  Needs no device.

    Where a tile's offsets would not fit 32 bits (rows of out 2^21 elements or more apart, of x 2^23 bytes, 256 rows of w, gated
    n + 256, over 2^32 - 2^16 bytes) no kernel with tiles is taken: "few" for up to 32 rows of x, else "any", which also takes all
    codes that are not 16-byte aligned."""
    plan = (ctypes.c_int64 * 2)()
    _lib.call("st_matmul_8bit_plan", m, k, n, int(gated), plan)
    return KERNELS[plan[0]], plan[1]


def matmul_8bit(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
                relu: bool = False, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """x [m, k] @ w [n, k]^T with both rows' scales, + bias (float32 [n]), then ReLU if asked: a Linear layer in 8 bits.

    Returns [m, n] in `dtype` (`out` if given, of that type).  Sums of codes (-127 to 127) are exact, k up to 131072; scales, bias and the
    one rounding to `dtype` follow.  Codes and out may have any row stride; codes whose rows are 16-byte aligned, as
    quantize_8bit lays them, are many times faster than others."""
    return _product("st_matmul_8bit", x, x_scales, w, w_scales, bias, int(bool(relu)), 1, dtype, out, stream)


def gated_8bit(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
               activation: str = "silu", dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """act(x @ gate^T) * (x @ up^T), both projections of a gated feed-forward layer in one launch: w [2n, k] holds the gate's
    rows, then the other's (w_scales and bias [2n] likewise); activation "silu" (g / (1 + exp(-g))) or "gelu" (g Phi(g)).

    Returns [m, n] in `dtype`; the rest is as for matmul_8bit."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation is one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return _product("st_gated_8bit", x, x_scales, w, w_scales, bias, ACTIVATIONS[activation], 2, dtype, out, stream)
