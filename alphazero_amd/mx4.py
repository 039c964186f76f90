"""4-bit floats with a power-of-two scale for every 32 (MX4): quantisation and a linear layer on them.

A row is cut into blocks of 32 along its last dimension; a block shares the scale 2^(floor(log2 max|x|) - 2), an element
is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (or its negative) times that scale, to nearest with ties to the even code, larger
ones to 6.  A block with an infinity or a NaN reads as NaN.  The matrix units multiply such numbers four times as fast
as halves, and a weight takes 4.25 bits.

    weight = mx4.quantize(layer.weight)                    # once
    y = mx4.linear(x, weight, bias=layer.bias, relu=True)  # x is quantised on the way in, sums are float32

The functions run on the tensors' device, on torch's current stream there; they wait for nothing and can be captured into
a graph.  They have no backward pass and refuse tensors that ask for one.  Engine(precision="mx4") evaluates the
network's linear layer with the same kernels.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Union

import torch

from . import _lib
from ._lib import Mx4LinearArgs, check
from ._tensors import dtype_code, no_grad, on_device, ptr, share_memory, stream_of

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
        self._take(codes, scales, shape, rows, cols)

    def _take(self, codes, scales, shape, rows, cols):
        self.codes, self.scales, self.shape, self._rows, self._cols = codes, scales, shape, rows, cols
        return self

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the codes stand for, rounded once to `dtype`."""
        with on_device(self.codes):
            out = torch.empty(self.shape, dtype=dtype, device=self.codes.device)
            code = dtype_code(out, "dtype")
            check(_lib.load().nnb_mx4_dequantize(stream_of(out), code, self._rows, self._cols, ptr(self.codes),
                                                 ptr(self.scales), ptr(out)), "nnb_mx4_dequantize")
        return out

    def __repr__(self):
        return f"MX4Tensor(shape={tuple(self.shape)}, device={self.device})"


def _rows_view(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, cols] without a copy where its strides allow one view."""
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
        units, device, (row_stride, col_stride) = _units(rows, cols), x.device, v.stride()
        codes = torch.empty(units + (4096,), dtype=torch.uint8, device=device)
        scales = torch.empty(units + (256,), dtype=torch.uint8, device=device)
        check(_lib.load().nnb_mx4_quantize(stream_of(x), code, rows, cols, ptr(v), row_stride, col_stride, ptr(codes),
                                           ptr(scales)), "nnb_mx4_quantize")
    return MX4Tensor.__new__(MX4Tensor)._take(codes, scales, x.shape, rows, cols)       # right by construction


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
    y_shape = tuple(x.shape[:-1]) + (n,)
    with on_device(weight.codes):
        if out is None:
            out = torch.empty(y_shape, dtype=out_dtype, device=device)
        elif tuple(out.shape) != y_shape or out.dtype != out_dtype:
            raise ValueError(f"out is {out.dtype} {tuple(out.shape)}, expected {out_dtype} {y_shape}")
        else:
            if any(t is not None and share_memory(out, t) for t in ((x.codes, x.scales) if quantized else (x,))
                   + (weight.codes, weight.scales, bias)):
                raise ValueError("out shares memory with an input")
            torch.autograd.graph.increment_version(out)              # the kernels write behind torch's back
        no_grad("mx4.linear", out)
        y_stride = n if out.is_contiguous() else _row_stride(out, n)
        args = Mx4LinearArgs()
        if quantized:
            rows = x._rows
            args.x_codes, args.x_scales = ptr(x.codes), ptr(x.scales)
        else:
            v = _rows_view(x)
            rows = v.shape[0]
            args.x = ptr(v)
            args.x_row_stride, args.x_col_stride = v.stride()
        args.rows, args.cols, args.out_features = rows, cols, n
        args.w_codes, args.w_scales = ptr(weight.codes), ptr(weight.scales)
        b = bias.contiguous() if bias is not None else None
        args.bias = ptr(b) if b is not None else None
        args.y, args.y_row_stride = ptr(out), y_stride
        args.x_type, args.y_type, args.relu = x_type, dtype_code(out, "out"), int(bool(relu))
        args.bias_type = dtype_code(bias, "bias") if bias is not None else 0
        nbytes = _workspace_bytes(rows, cols, n, quantized)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        check(_lib.load().nnb_mx4_linear(stream_of(out), C.byref(args), ptr(workspace) if nbytes else None, nbytes),
              "nnb_mx4_linear")
    return out
