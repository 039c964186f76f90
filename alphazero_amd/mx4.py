"""4-bit floats with a power-of-two scale for every 32 (MX4): quantisation and a linear layer on them.

A row is cut into blocks of 32 along its last dimension; a block shares the scale 2^(floor(log2 max|x|) - 2), an element
is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (or its negative) times that scale, to nearest with ties to the even code, larger
ones to 6.  A block with an infinity or a NaN reads as NaN.  The matrix units multiply such numbers four times as fast
as halves, and a weight takes 4.25 bits.

    with torch.no_grad():
        weight = mx4.quantize(layer.weight)                    # once
        y = mx4.linear(x, weight, bias=layer.bias, relu=True)  # x is quantised on the way in, sums are float32

The functions run on the tensors' device, on torch's current stream there; they wait for nothing and can be captured into
a graph.  They have no derivatives and refuse tensors that ask for a backward pass or carry a forward-mode tangent.
Engine(precision="mx4") evaluates the network's linear layer with the same kernels.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Union

import torch

from . import _lib
from ._lib import Mx4LinearArgs, check
from ._tensors import DTYPES, dtype_code, no_grad, on_device, resolved, share_memory, stream_of, writable

BLOCK = 32                              # elements that share a scale
UNIT_ROWS, UNIT_COLS = 32, 256          # rows and columns are padded with zeros to whole units


def _units(rows: int, cols: int) -> tuple:
    return -(-rows // UNIT_ROWS), -(-cols // UNIT_COLS)


class MX4Tensor:
    """Quantised numbers of shape `shape`, blocks along the last dimension.

    Units of 32 rows x 256 columns (include/nnb.h gives the order within, the matrix instructions'):
    codes   uint8 [ceil(rows/32), ceil(cols/256), 4096]
    scales  uint8 [ceil(rows/32), ceil(cols/256), 256], exponent + 127, 255 = not a number
    """

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape):
        shape = torch.Size(shape)
        if len(shape) < 1 or shape[-1] < 1:
            raise ValueError(f"shape {tuple(shape)} has no last dimension to cut into blocks")
        rows, cols = shape[:-1].numel(), shape[-1]
        units = _units(rows, cols)
        for name, t, want in (("codes", codes, units + (4096,)), ("scales", scales, units + (256,))):
            if t.dtype != torch.uint8 or tuple(t.shape) != want or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous uint8 of shape {want}, got {t.dtype} {tuple(t.shape)}")
        if codes.device != scales.device:
            raise ValueError("codes and scales are on different devices")
        self.shape, self.device, self._rows, self._cols, self._units = shape, codes.device, rows, cols, units
        self._codes, self._scales = codes, scales

    @classmethod
    def _of_buffer(cls, buffer, shape, rows, cols, units):
        """All codes, then all scales in one allocation; the two tensors are made when somebody asks for them."""
        self = cls.__new__(cls)
        self.shape, self.device, self._rows, self._cols, self._units = shape, buffer.device, rows, cols, units
        self._codes, self._scales, self._buffer = None, None, buffer
        return self

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._buffer[:self._units[0] * self._units[1] * 4096].view(self._units + (4096,))
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._buffer[self._units[0] * self._units[1] * 4096:].view(self._units + (256,))
        return self._scales

    def _pointers(self) -> tuple:
        if self._codes is None or self._scales is None:
            base = self._buffer.data_ptr()
            return base, base + self._units[0] * self._units[1] * 4096
        return self._codes.data_ptr(), self._scales.data_ptr()

    def _tensors(self) -> tuple:
        return (self._buffer,) if self._codes is None else (self.codes, self.scales)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the codes stand for, rounded once to `dtype`."""
        if dtype not in DTYPES:
            raise ValueError(f"dtype is {dtype}: expected float32, float16 or bfloat16")
        with on_device(self):
            out = torch.empty(self.shape, dtype=dtype, device=self.device)
            codes, scales = self._pointers()
            check(_lib.load().nnb_mx4_dequantize(stream_of(out), DTYPES[dtype], self._rows, self._cols, codes, scales,
                                                 out.data_ptr()), "nnb_mx4_dequantize")
        return out

    def __repr__(self):
        return f"MX4Tensor(shape={tuple(self.shape)}, device={self.device})"


def _rows_view(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, cols] without a copy where its strides allow one view."""
    if x.is_neg():
        x = resolved(x)
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


def _row_stride(out: torch.Tensor, n: int) -> int:
    """Elements between consecutive rows of n contiguous elements of `out`."""
    if out.numel() == 0:
        return n
    try:
        y = out.view(-1, n)
    except RuntimeError:
        raise ValueError(f"out of shape {tuple(out.shape)}, strides {out.stride()} is no matrix of evenly spaced rows") from None
    if (n > 1 and y.stride(1) != 1) or (y.shape[0] > 1 and y.stride(0) < n):
        raise ValueError("out must have contiguous rows that do not overlap")
    return max(y.stride(0), n)


def quantize(x: torch.Tensor) -> MX4Tensor:
    """x (float32, float16 or bfloat16, at least one dimension, any strides) -> MX4Tensor of the same shape."""
    code = dtype_code(x, "x")
    no_grad("mx4.quantize", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x of shape {tuple(x.shape)} has no last dimension to cut into blocks")
    with on_device(x):
        v = _rows_view(x)
        rows, cols = v.shape
        units, (row_stride, col_stride) = _units(rows, cols), v.stride()
        count = units[0] * units[1]
        buffer = torch.empty(count * (4096 + 256), dtype=torch.uint8, device=x.device)
        codes = buffer.data_ptr()
        check(_lib.load().nnb_mx4_quantize(stream_of(x), code, rows, cols, v.data_ptr(), row_stride, col_stride, codes,
                                           codes + count * 4096), "nnb_mx4_quantize")
    return MX4Tensor._of_buffer(buffer, x.shape, rows, cols, units)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(rows: int, cols: int, n: int, quantized: bool) -> int:
    nbytes = C.c_size_t()
    check(_lib.load().nnb_mx4_linear_workspace_bytes(rows, cols, n, int(quantized), C.byref(nbytes)),
          "nnb_mx4_linear_workspace_bytes")
    return nbytes.value


def linear(x: Union[torch.Tensor, MX4Tensor], weight: MX4Tensor, bias: Optional[torch.Tensor] = None, relu: bool = False,
           out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., K] times weight [N, K] transposed, plus bias [N], then ReLU if asked: [..., N].

    x may be numbers (quantised inside the call) or an MX4Tensor.  Products are exact, sums, bias and ReLU in float32,
    one rounding to `out_dtype` (default: x's type, float32 for an MX4Tensor).  `out` ([..., N], rows contiguous, no
    element in common with the inputs) is written instead of a new tensor when given."""
    if not isinstance(weight, MX4Tensor) or len(weight.shape) != 2:
        raise ValueError("weight must be a two-dimensional MX4Tensor (mx4.quantize)")
    quantized = isinstance(x, MX4Tensor)
    n, cols = weight.shape
    if len(x.shape) < 1 or x.shape[-1] != cols:
        raise ValueError(f"x of shape {tuple(x.shape)} does not fit a weight of shape {tuple(weight.shape)}")
    if not quantized:
        x_type = dtype_code(x, "x")
        no_grad("mx4.linear", x, bias)
    else:
        x_type = 0
        no_grad("mx4.linear", bias)
    device = weight.device
    if x.device != device or (bias is not None and bias.device != device) or (out is not None and out.device != device):
        raise ValueError("x, weight, bias and out must be on one device")
    if bias is not None and (tuple(bias.shape) != (n,)):
        raise ValueError(f"bias of shape {tuple(bias.shape)}, expected {(n,)}")
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else torch.float32 if quantized else x.dtype
    if out is not None:
        writable(out, "out")
        no_grad("mx4.linear", out)
    y_shape = tuple(x.shape[:-1]) + (n,)
    with on_device(weight):
        if out is None:
            out = torch.empty(y_shape, dtype=out_dtype, device=device)
            y_stride = n
        else:
            if tuple(out.shape) != y_shape or out.dtype != out_dtype:
                raise ValueError(f"out is {out.dtype} {tuple(out.shape)}, expected {out_dtype} {y_shape}")
            y_stride = n if out.is_contiguous() else _row_stride(out, n)
            for t in (x._tensors() if quantized else (x,)) + weight._tensors() + (() if bias is None else (bias,)):
                if share_memory(out, t):
                    raise ValueError("out shares memory with an input")
            torch.autograd.graph.increment_version(out)              # the kernels write behind torch's back
        if quantized:
            rows, x_ptr, row_stride, col_stride = x._rows, None, 0, 0
            x_codes, x_scales = x._pointers()
        else:
            v = _rows_view(x)
            rows, x_ptr, x_codes, x_scales = v.shape[0], v.data_ptr(), None, None
            row_stride, col_stride = v.stride()
        w_codes, w_scales = weight._pointers()
        b = None if bias is None else resolved(bias).contiguous()
        y_type = dtype_code(out, "out")
        bias_type, b_ptr = (0, None) if b is None else (dtype_code(b, "bias"), b.data_ptr())
        args = Mx4LinearArgs(rows, cols, n, x_ptr, row_stride, col_stride, x_codes, x_scales, w_codes, w_scales, b_ptr,
                             out.data_ptr(), y_stride, x_type, bias_type, y_type, int(bool(relu)))
        nbytes = _workspace_bytes(rows, cols, n, quantized)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        check(_lib.load().nnb_mx4_linear(stream_of(out), C.byref(args), workspace.data_ptr() if nbytes else None, nbytes),
              "nnb_mx4_linear")
    return out
