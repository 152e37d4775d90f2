"""4-bit weights on MI355X: the quantiser and the Linear layer of a decoding step (no reference counterpart; the
weights are held as the 2-bit store holds its keys, codes and f32 scales, with a lowest value beside each scale).

A group of `group` weights along k has lo = min, hi = max and scale = (hi - lo) / 15; a weight is held as
code = round_half_even((w - lo) * 15 / (hi - lo)), decided in 64 bits, and stands for scale * code + lo.  Code i is in
byte i // 2, bits 4 * (i % 2).  A group that holds a NaN or an infinity reads as NaN throughout.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .matmul import _stream

GROUPS = (32, 64, 128)
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # ST_F32, ST_F16, ST_BF16


def _dtype(t: torch.Tensor, what: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} is a torch tensor")
    if t.dtype not in DTYPES:
        raise ValueError(f"{what} is {t.dtype}; float32, float16 and bfloat16 are taken")
    return DTYPES[t.dtype]


def _rows(t: torch.Tensor, what: str) -> int:
    """Elements from a row to the next of a [rows, ...] tensor whose rows are contiguous."""
    shape, strides = t.shape, t.stride()
    width = 1
    for size in shape[1:]:
        width *= size
    if not shape[0] or t.is_contiguous():
        return width
    run = 1
    for size, stride in zip(reversed(shape[1:]), reversed(strides[1:])):
        if size != 1 and width and stride != run:
            raise ValueError(f"{what} has rows that are not contiguous (shape {list(shape)}, strides {list(strides)})")
        run *= size
    if shape[0] > 1 and strides[0] < run:
        raise ValueError(f"{what} has rows that overlap (shape {list(shape)}, strides {list(strides)})")
    return strides[0] if shape[0] > 1 else run


def _plain(t: torch.Tensor, dtype: torch.dtype, shape, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} is a torch tensor")
    if t.dtype != dtype or not t.is_contiguous() or t.shape != shape:
        raise ValueError(f"{what} is a contiguous {dtype} tensor {list(shape)}; got {t.dtype} {list(t.shape)}"
                         + ("" if t.is_contiguous() else " that is not contiguous"))
    return t


def _extent(t: torch.Tensor) -> Tuple[int, int]:
    """The first byte of a tensor and the one behind its last."""
    start = t.data_ptr()
    if t.is_contiguous():
        return start, start + t.nbytes
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return start, start + (last + 1) * t.element_size()


def _apart(outs, ins) -> None:
    """No output shares memory with an input or with another output; (tensor or None, name) pairs."""
    spans = []
    for pairs, out in ((outs, True), (ins, False)):
        for t, name in pairs:
            if t is not None:
                a, b = _extent(t)
                if a < b:
                    spans.append((a, b, out, name))
    spans.sort()
    # By their starts: an output may not start before the end of anything earlier, an input not before an output's.
    end = out_end = 0
    for a, b, out, name in spans:
        if a < (end if out else out_end):
            other = next(o for c, d, other_out, o in spans if c <= a < d and o != name and (out or other_out))
            raise ValueError(f"{name} shares memory with {other}" if out else f"{other} shares memory with {name}")
        if b > end:
            end = b
        if out and b > out_end:
            out_end = b


def _on_gpu(first: torch.Tensor, tensors) -> None:
    """Every given tensor on the GPU of the first."""
    if not first.is_cuda:
        raise ValueError("tensors live on the GPU")
    index = first.get_device()
    for t, name in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, the rest on {first.device}")


class _launch:
    """Makes `device` current and, inside, gives the handle of the stream to launch on (the device's current one if
    `stream` is None); what is allocated inside belongs to that stream."""
    __slots__ = ("device", "stream", "inside")

    def __init__(self, device: torch.device, stream):
        self.device, self.stream, self.inside = device, stream, None

    def __enter__(self) -> int:
        if self.stream is None and torch.cuda.current_device() == self.device.index:
            return _stream(None)
        with contextlib.ExitStack() as stack:
            stack.enter_context(torch.cuda.device(self.device))
            handle = _stream(self.stream)
            if self.stream is not None and handle != _stream(None):
                stack.enter_context(torch.cuda.stream(torch.cuda.ExternalStream(handle, device=self.device)))
            self.inside = stack.pop_all()
        return handle

    def __exit__(self, *error) -> None:
        if self.inside is not None:
            self.inside.__exit__(*error)


def _addr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def quantize_4bit(x: torch.Tensor, group: int = 128, values: Union[bool, torch.Tensor] = False, stream=None):
    """Weights x [n, k] (any row stride) -> codes [n, k/2] uint8 and scales [n, k/group, 2] float32 (scale, lo).

    values: also return what the codes stand for, [n, k] in x's type (True: a new tensor, or a tensor to fill), the
    forward value of a straight-through gradient."""
    dtype = _dtype(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x is [n, k], got {list(x.shape)}")
    n, k = x.shape
    if group not in GROUPS:
        raise ValueError(f"group is one of {GROUPS}, got {group}")
    if k == 0 or k % group:
        raise ValueError(f"k = {k} is not a multiple of the group, {group}")
    stride = _rows(x, "x")
    out = values if isinstance(values, torch.Tensor) else None
    if out is not None:
        _plain(out, x.dtype, (n, k), "values")
        _apart([(out, "values")], [(x, "x")])
    _on_gpu(x, [(out, "values")])
    with _launch(x.device, stream) as handle:
        codes = torch.empty((n, k // 2), dtype=torch.uint8, device=x.device)
        scales = torch.empty((n, k // group, 2), dtype=torch.float32, device=x.device)
        if out is None and values:
            out = torch.empty((n, k), dtype=x.dtype, device=x.device)
        _lib.call("st_quantize_4bit", x.data_ptr(), dtype, n, k, stride, group, codes.data_ptr(), scales.data_ptr(),
                  _addr(out), handle)
    return (codes, scales) if out is None else (codes, scales, out)


def matvec_4bit(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
                relu: bool = False, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """x [m, k] @ w^T + bias, then ReLU if asked, for 4-bit weights w [n, k] (codes and scales of quantize_4bit): the
    Linear layer of a decoding step.  Returns [m, n] in x's type (`out` if given); x and out may have any row stride,
    bias is float32 [n].  For large m, a product over `values` of quantize_4bit is faster."""
    dtype = _dtype(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x is [m, k], got {list(x.shape)}")
    m, k = x.shape
    if not isinstance(codes, torch.Tensor) or codes.dim() != 2 or codes.shape[1] * 2 != k:
        raise ValueError(f"codes are [n, {k // 2}] for x {list(x.shape)}")
    n = codes.shape[0]
    _plain(codes, torch.uint8, (n, k // 2), "codes")
    if not isinstance(scales, torch.Tensor) or scales.dim() != 3 or scales.shape[1] == 0 or k % scales.shape[1]:
        raise ValueError("scales are [n, k / group, 2]")
    group = k // scales.shape[1]
    if group not in GROUPS:
        raise ValueError(f"scales {list(scales.shape)} of k = {k} have groups of {group}; they are of one of {GROUPS}")
    _plain(scales, torch.float32, (n, k // group, 2), "scales")
    if bias is not None:
        _plain(bias, torch.float32, (n,), "bias")
    stride = _rows(x, "x")
    if out is not None:
        if _dtype(out, "out") != dtype or tuple(out.shape) != (m, n):
            raise ValueError(f"out is {x.dtype} [{m}, {n}]; got {out.dtype} {list(out.shape)}")
        _rows(out, "out")
        _apart([(out, "out")], [(x, "x"), (codes, "codes"), (scales, "scales"), (bias, "bias")])
    _on_gpu(x, [(codes, "codes"), (scales, "scales"), (bias, "bias"), (out, "out")])
    with _launch(x.device, stream) as handle:
        if out is None:
            out = torch.empty((m, n), dtype=x.dtype, device=x.device)
        _lib.call("st_matvec_4bit", x.data_ptr(), dtype, m, k, stride, codes.data_ptr(), scales.data_ptr(), group, n,
                  _addr(bias), int(bool(relu)), out.data_ptr(), _rows(out, "out"), handle)
    return out
