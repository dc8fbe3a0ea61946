"""Microscaled formats on the HIP kernels: quantisation and the product of a quantised linear.

* ``quantize`` / ``dequantize``  -> ``mpq_mx_quantize`` / ``mpq_mx_dequantize``
* ``linear``                     -> ``mpq_mx_linear``: ``Q(x) W^T + bias`` on the scaled matrix products

A block is 32 consecutive values of the last dimension with one power-of-two scale
``2^(floor(log2(max |x|)) - emax)``, held as its biased exponent in one byte.  ``mxfp4`` holds E2M1 values
(0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives; emax 2), ``mxfp8`` E4M3 values (up to 448; emax 8).
Values are rounded to nearest, ties to even, and saturate.  A block with a NaN or an infinity reads back as NaN.
No counterpart in the reference, whose formats are integer grids and the E8P12 codebook.

Tensors live on the ROCm device; there is no CPU path, and no gradient: a backward pass through a result raises.
"""
from __future__ import annotations

import math
import operator
from typing import Optional, Tuple, Union

import torch

from . import _lib, ops

FORMATS = {"mxfp4": 0, "mxfp8": 1}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BLOCK = 32
ROW = 256  # rows of codes are padded with zeros to whole 256-value pieces


def _fmt(fmt: str) -> int:
    try:
        return FORMATS[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"unknown microscaled format {fmt!r}; expected 'mxfp4' or 'mxfp8'") from None


def _dtype(t: torch.dtype, what: str) -> int:
    if t not in DTYPES:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t}")
    return DTYPES[t]


def padded(cols: int) -> int:
    """Values of a row of codes with its padding."""
    return (int(cols) + ROW - 1) // ROW * ROW


def code_bytes(cols: int, fmt: str) -> int:
    """Bytes of a row of codes."""
    return padded(cols) // (2 if _fmt(fmt) == 0 else 1)


def _on_device(*ts: Optional[torch.Tensor]) -> torch.device:
    dev = ts[0].device
    if dev.type != "cuda":
        raise ValueError(f"mpq_amd operates on ROCm device tensors only (got a tensor on {dev}).")
    for t in ts[1:]:
        if t is not None and t.device != dev:
            raise ValueError("all tensors must be on the same device")
    return dev


class _NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, name, out, x, bias):
        ctx.name = name
        ctx.mark_dirty(out)
        return out

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no gradient")


def _no_gradient(name: str, out: torch.Tensor, x: Optional[torch.Tensor],
                 bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out``, through which a backward pass raises if gradients of ``x`` or ``bias`` are recorded."""
    if (x is not None and x.requires_grad or bias is not None and bias.requires_grad) and torch.is_grad_enabled():
        return _NoGradient.apply(name, out, x, bias)
    return out


class MXTensor:
    """A quantised tensor: ``codes`` (rows, :func:`code_bytes`) and ``scales`` (rows, padded cols / 32), both uint8.

    ``cols`` is the length of the last dimension; ``lead`` the other ones (``rows`` is their product).  In ``mxfp4``
    a byte holds two codes, the first in its low half.  Codes behind ``cols`` are zero.  The attributes are checked
    once and cannot be replaced (their contents may change)."""

    __slots__ = ("_codes", "_scales", "_cols", "_fmt", "_lead", "_rows", "_device", "_f")
    codes, scales, cols, fmt, lead, rows, device = (
        property(operator.attrgetter("_" + n)) for n in ("codes", "scales", "cols", "fmt", "lead", "rows", "device"))

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int, fmt: str = "mxfp4",
                 lead: Optional[Tuple[int, ...]] = None) -> None:
        cols, f = int(cols), _fmt(fmt)
        if cols < 1:
            raise ValueError(f"cols must be >= 1, got {cols}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2:
            raise ValueError("codes and scales must be 2-D uint8 tensors")
        rows, width = codes.shape
        wide = padded(cols)
        if width != (wide // 2 if f == 0 else wide) or scales.shape != (rows, wide // BLOCK):
            raise ValueError(f"{fmt} rows of {cols} values need codes ({rows}, {code_bytes(cols, fmt)}) and scales "
                             f"({rows}, {wide // BLOCK}); got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise ValueError("codes and scales must be contiguous and 16-byte aligned")
        lead = (rows,) if lead is None else tuple(int(n) for n in lead)
        if math.prod(lead) != rows:
            raise ValueError(f"leading dimensions {lead} do not make {rows} rows")
        self._set(codes, scales, cols, fmt, f, lead, rows, _on_device(codes, scales))

    def _set(self, codes, scales, cols, fmt, f, lead, rows, device) -> "MXTensor":
        self._codes, self._scales, self._cols, self._fmt, self._f = codes, scales, cols, fmt, f
        self._lead, self._rows, self._device = lead, rows, device
        return self

    @property
    def shape(self) -> Tuple[int, ...]:
        return (*self._lead, self._cols)


def _rows(x: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """(x as rows with a contiguous last dimension, its row stride); a copy only where its strides are otherwise."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    rows, cols = x.shape
    ld, step = x.stride()
    if (step != 1 and cols > 1) or (ld < cols and rows > 1):
        return x.contiguous(), cols
    return x, ld if rows > 1 else cols


def quantize(x: torch.Tensor, fmt: str = "mxfp4") -> MXTensor:
    """Quantise along the last dimension (any length; a short last block counts only its values)."""
    f, dt = _fmt(fmt), _dtype(x.dtype, "x")
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"x needs a last dimension of at least 1, got {tuple(shape)}")
    dev = _on_device(x)
    cols = shape[-1]
    rows = math.prod(shape[:-1])
    wide = padded(cols)
    codes = torch.empty((rows, wide // 2 if f == 0 else wide), dtype=torch.uint8, device=dev)
    scales = torch.empty((rows, wide // BLOCK), dtype=torch.uint8, device=dev)
    if rows:
        x, ld = _rows(x)
        with ops.on_device(dev):
            _lib.check(_lib.load().mpq_mx_quantize(x.data_ptr(), dt, rows, cols, ld, f, codes.data_ptr(),
                                                   scales.data_ptr(), ops.raw_stream(dev)), "mpq_mx_quantize")
    return MXTensor.__new__(MXTensor)._set(codes, scales, cols, fmt, f, tuple(shape[:-1]), rows, dev)


def dequantize(t: MXTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that ``t`` stands for (exact in float32 and bfloat16)."""
    dt, dev = _dtype(dtype, "dtype"), t._device
    out = torch.empty(t.shape, dtype=dtype, device=dev)
    if t._rows:
        with ops.on_device(dev):
            _lib.check(_lib.load().mpq_mx_dequantize(t._codes.data_ptr(), t._scales.data_ptr(), t._rows, t._cols, t._f,
                                                     out.data_ptr(), dt, t._cols, ops.raw_stream(dev)),
                       "mpq_mx_dequantize")
    return out


def linear(x: Union[torch.Tensor, MXTensor], weight: MXTensor, bias: Optional[torch.Tensor] = None, *,
           act_format: str = "mxfp4", dtype: Optional[torch.dtype] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``Q(x) weight^T + bias`` over the last dimension.

    ``weight`` (out features x in features) is ``mxfp4``.  ``x`` is quantised to ``act_format`` within the call, or
    comes as an :class:`MXTensor` in either format.  The result has ``dtype`` (default: that of ``x``; bfloat16 for an
    :class:`MXTensor`); ``out`` (contiguous, of that shape and type) receives it in place of a new tensor.

    A backward pass through the result raises (a given ``out`` is left out of it).

    Sums are held in fp32.  With ``mxfp8`` the matrix core cuts the terms of each 32-value block at 2^-13 of the
    block's largest product, some 1e-4 of the result: fine for 16-bit results, and less than the format's own error."""
    if weight._f != 0 or len(weight._lead) != 1:
        raise ValueError("weight must be a 2-D mxfp4 MXTensor (out features x in features)")
    given, fresh = isinstance(x, MXTensor), out is None
    f = x._f if given else _fmt(act_format)
    shape, rows, cols = x.shape, weight._rows, weight._cols
    if len(shape) < 1 or shape[-1] != cols:
        raise ValueError(f"x has shape {tuple(shape)}, weight takes {cols} features")
    dev = _on_device(weight._codes, x._codes if given else x, bias, out)
    if dtype is None:
        dtype = out.dtype if out is not None else torch.bfloat16 if given else x.dtype
    odt = _dtype(dtype, "dtype")
    xdt = 0 if given else _dtype(x.dtype, "x")
    if bias is not None:
        if bias.shape != (rows,):
            raise ValueError(f"bias must have shape ({rows},), got {tuple(bias.shape)}")
        bias = ops._f32c(bias)
    shape = (*shape[:-1], rows)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
    elif out.shape != shape or out.dtype != dtype or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {dtype} tensor of shape {shape}")
    tokens = math.prod(shape[:-1])
    if tokens == 0 or rows == 0:
        return out
    lib = _lib.load()
    if given:
        src = (None, 0, cols, x._codes.data_ptr(), x._scales.data_ptr())
    else:
        x, ld = _rows(x)
        src = (x.data_ptr(), xdt, ld, None, None)
    need = lib.mpq_mx_linear_workspace_size(tokens, cols, rows, f)
    ws = ops.workspace(need, dev) if need else None
    with ops.on_device(dev):
        _lib.check(lib.mpq_mx_linear(*src, f, tokens, cols, weight._codes.data_ptr(), weight._scales.data_ptr(), rows,
                                     None if bias is None else bias.data_ptr(), out.data_ptr(), odt, rows,
                                     None if ws is None else ws.data_ptr(), need, ops.raw_stream(dev)),
                   "mpq_mx_linear")
    if fresh and (bias is not None or not given and x.requires_grad):
        return _no_gradient("mx.linear", out, None if given else x, bias)
    return out
