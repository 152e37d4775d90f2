"""Row kernels on MI355X: causal softmax and its backward (gpu_step/rows.rs:101-123),
LayerNorm forward and backward (gpu_step/rows.rs:60-99); the root-mean-square norm with the residual's addition, its 8-bit
rows and its backward (no reference counterpart)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .matmul import _ptr, _stream
from .quant4 import DTYPES, _addr, _dtype, _launch, _on_gpu, _plain, _rows
from .quant8 import _new_codes


def _check_rows_out(out: torch.Tensor | None, n: int, device, name: str) -> None:
    """A caller-supplied output must hold every element the kernel writes (rows x n floats) on the input's
    device."""
    if out is None:
        return
    if out.numel() < n:
        raise ValueError(f"{name}: out holds {out.numel()} elements, the call writes {n}")
    if out.device != device:
        raise ValueError(f"{name}: out is on {out.device}, the input on {device}")


def softmax(x: torch.Tensor, rows: int, n: int, t: int, scale: float, causal: bool, one: bool,
            out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Row-wise softmax of scale*x over x [rows, n] (rows.rs:101-112); returns y."""
    _check_rows_out(out, rows * n, x.device, "softmax")
    y = out if out is not None else torch.empty(rows * n, dtype=torch.float32, device=x.device)
    _lib.call("st_softmax", _ptr(x), _ptr(y), rows, n, t, float(scale), int(causal), int(one), _stream(stream))
    return y


def softmax_backward(dy: torch.Tensor, y: torch.Tensor, rows: int, n: int, scale: float,
                     out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """dx = scale * y * (dy - sum(dy * y)) per row (rows.rs:114-123); returns dx."""
    _check_rows_out(out, rows * n, y.device, "softmax_backward")
    dx = out if out is not None else torch.empty(rows * n, dtype=torch.float32, device=y.device)
    _lib.call("st_softmax_backward", _ptr(dy), _ptr(y), _ptr(dx), rows, n, float(scale), _stream(stream))
    return dx


@dataclass
class LnOut:
    """What LayerNorm's backward needs from its forward (rows.rs:52-58)."""
    y: torch.Tensor
    mean: torch.Tensor
    rstd: torch.Tensor


def layer_norm(x: torch.Tensor, rows: int, d: int, params: torch.Tensor, off: int, eps: float = 1e-5,
               models: int = 1, model_stride: int = 0, stream=None) -> LnOut:
    """y = (x - mean) / sqrt(var + eps) * gamma + beta per row (rows.rs:65); gamma, beta at params[off..]."""
    dev = x.device
    out = LnOut(torch.empty(rows * d, dtype=torch.float32, device=dev), torch.empty(rows, dtype=torch.float32, device=dev),
                torch.empty(rows, dtype=torch.float32, device=dev))
    _lib.call("st_layer_norm", _ptr(x), rows, d, _ptr(params), off, float(eps), models, model_stride, _ptr(out.y),
              _ptr(out.mean), _ptr(out.rstd), _stream(stream))
    return out


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, fwd: LnOut, rows: int, d: int, params: torch.Tensor,
                        grads: torch.Tensor, off: int, dx: torch.Tensor, accumulate: bool, models: int = 1,
                        model_stride: int = 0, stream=None) -> None:
    """dx (+)= LayerNorm's input gradient; gamma / beta gradients accumulate into grads at off (rows.rs:90)."""
    _lib.call("st_layer_norm_backward", _ptr(dy), _ptr(x), _ptr(fwd.mean), _ptr(fwd.rstd), rows, d, _ptr(params),
              _ptr(grads), off, _ptr(dx), int(accumulate), models, model_stride, _stream(stream))


@dataclass
class RmsOut:
    """What rms_norm returns: h, the rows it normed (x + residual, or x itself); of y, rstd [rows] float32 (with y, and for the
    backward pass), codes, scales and values what was asked for."""
    h: torch.Tensor
    rstd: Optional[torch.Tensor] = None
    y: Optional[torch.Tensor] = None
    codes: Optional[torch.Tensor] = None
    scales: Optional[torch.Tensor] = None
    values: Optional[torch.Tensor] = None


def _norm_rows(t: torch.Tensor, like: torch.Tensor, what: str) -> int:
    """The row stride of a [rows, d] tensor of another's shape and type."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} is a torch tensor")
    if t.dtype != like.dtype or t.shape != like.shape:
        raise ValueError(f"{what} is {like.dtype} {list(like.shape)}; got {t.dtype} {list(t.shape)}")
    return _rows(t, what)


def _norm_weight(weight: torch.Tensor, x: torch.Tensor) -> int:
    if not isinstance(weight, torch.Tensor):
        raise TypeError("weight is a torch tensor")
    if weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"weight is float32 or of the rows' type, {x.dtype}; got {weight.dtype}")
    _plain(weight, weight.dtype, (x.shape[1],), "weight")
    return DTYPES[weight.dtype]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-5, y: bool = True,
             eight_bit: bool = False, values: bool = False, stream=None, *, rstd: bool = False) -> RmsOut:
    """h = x + residual (x itself without one), rounded to x's type, and its norm h / sqrt(mean h^2 + eps) * weight per row of
    x [rows, d] (float32, float16 or bfloat16, any row stride); weight [d] is of x's type or float32.

    y: return the norm in x's type, and rstd with it.  eight_bit: return it as 8-bit rows for quant8's products, codes and scales, and with
    `values` also what those stand for in x's type.  The codes are those of the rows h * weight (1 / rms is a factor of a
    row's scale).  rstd: return it without y too, for the backward pass of who trains through `values`."""
    dtype = _dtype(x, "x")
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"x is [rows, d] with d > 0, got {list(x.shape)}")
    n, d = x.shape
    stride, w_dtype = _rows(x, "x"), _norm_weight(weight, x)
    r_stride = 0 if residual is None else _norm_rows(residual, x, "residual")
    if not eps >= 0:
        raise ValueError(f"eps is {eps}")
    if values and not eight_bit:
        raise ValueError("values are those of 8-bit rows: eight_bit=True")
    if not y and not eight_bit:
        raise ValueError("neither y nor 8-bit rows are asked for")
    _on_gpu(x, [(weight, "weight"), (residual, "residual")])
    with _launch(x.device, stream) as handle:
        h = x if residual is None else x.new_empty((n, d))
        out = codes = scales = stood = None
        if y:
            out = x.new_empty((n, d))
        inverse = x.new_empty((n,), dtype=torch.float32) if y or rstd else None
        if eight_bit:
            codes, scales = _new_codes(n, d, x), x.new_empty((n,), dtype=torch.float32)
            stood = x.new_empty((n, d)) if values else None
        _lib.call("st_rms_norm", x.data_ptr(), _addr(residual), dtype, n, d, stride, r_stride, weight.data_ptr(), w_dtype, eps,
                  0 if residual is None else h.data_ptr(), _addr(inverse), _addr(out), _addr(codes), (d + 15) // 16 * 16, _addr(scales),
                  _addr(stood), handle)
    return RmsOut(h, inverse, out, codes, scales, stood)


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor, dh: Optional[torch.Tensor] = None,
                      stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of rms_norm's y from dy, with h and rstd that it returned: dx [rows, d], the gradient of x and of the residual
    alike, in the rows' type, and the weight's [d], float32.  dh: the gradient that reaches h by other ways (the residual
    stream's), added to dx."""
    dtype = _dtype(h, "h")
    if h.dim() != 2 or h.shape[1] == 0:
        raise ValueError(f"h is [rows, d] with d > 0, got {list(h.shape)}")
    n, d = h.shape
    stride, w_dtype = _rows(h, "h"), _norm_weight(weight, h)
    dy_stride, dh_stride = _norm_rows(dy, h, "dy"), 0 if dh is None else _norm_rows(dh, h, "dh")
    _plain(rstd, torch.float32, (n,), "rstd")
    _on_gpu(h, [(dy, "dy"), (dh, "dh"), (rstd, "rstd"), (weight, "weight")])
    with _launch(h.device, stream) as handle:
        dx, dweight = h.new_empty((n, d)), h.new_empty((d,), dtype=torch.float32)
        need = _lib.lib().st_rms_norm_backward_bytes(n, d, dtype)
        work = h.new_empty((need,), dtype=torch.uint8) if need else None
        _lib.call("st_rms_norm_backward", dy.data_ptr(), h.data_ptr(), _addr(dh), dtype, n, d, dy_stride, stride, dh_stride, rstd.data_ptr(),
                  weight.data_ptr(), w_dtype, dx.data_ptr(), dweight.data_ptr(), _addr(work), need, handle)
    return dx, dweight
