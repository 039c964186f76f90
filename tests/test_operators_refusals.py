"""What the matrix operators refuse, checked without a GPU: bad arguments come back as errors before anything runs."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from alphazero_amd import _lib
    return _lib.load()


def _message(lib):
    return lib.nnb_last_error().decode()


def test_mx4_struct_matches_the_header(tmp_path):
    import os
    import subprocess
    from alphazero_amd import _lib
    from conftest import ROOT
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "nnb.h"\nint main(void){printf("%zu\\n",sizeof(nnb_mx4_linear_args));return 0;}\n')
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    assert int(subprocess.check_output([str(tmp_path / "s")])) == C.sizeof(_lib.Mx4LinearArgs)


def test_mx4_quantize_refuses_bad_arguments(lib):
    p = C.c_void_p(4096)                     # never read: every call below is refused or empty
    good = dict(t=0, rows=2, cols=64, x=p, codes=p, scales=p)
    def call(**kw):
        a = {**good, **kw}
        return lib.nnb_mx4_quantize(None, a["t"], a["rows"], a["cols"], a["x"], a["cols"], 1, a["codes"], a["scales"])
    for kw, word in ((dict(t=3), "dtype"), (dict(t=-1), "dtype"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"),
                     (dict(cols=0), "columns"), (dict(cols=(1 << 24) + 1), "columns"), (dict(x=None), "null"),
                     (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(codes=C.c_void_p(4100)), "aligned"),
                     (dict(scales=C.c_void_p(4097)), "aligned")):
        assert call(**kw) == -1 and word in _message(lib), kw
    assert call(rows=0, x=None) == 0
    assert lib.nnb_mx4_dequantize(None, 5, 2, 64, p, p, p) == -1
    assert lib.nnb_mx4_dequantize(None, 0, 2, 64, p, p, None) == -1


def test_mx4_linear_refuses_bad_arguments(lib):
    from alphazero_amd._lib import Mx4LinearArgs
    def call(ws=C.c_void_p(4096), ws_bytes=1 << 20, **kw):
        a = Mx4LinearArgs()
        base = dict(rows=4, cols=64, out_features=8, x=4096, x_row_stride=64, x_col_stride=1, w_codes=4096, w_scales=4096,
                    y=4096, y_row_stride=8)
        for k, v in {**base, **kw}.items():
            setattr(a, k, v)
        return lib.nnb_mx4_linear(None, C.byref(a), ws, ws_bytes)
    for kw, word in ((dict(rows=-1), "rows"), (dict(cols=0), "columns"), (dict(x_type=9), "x_type"), (dict(y_type=9), "y_type"),
                     (dict(bias=4096, bias_type=9), "bias_type"), (dict(w_codes=None), "null"), (dict(y=None), "null"),
                     (dict(x=None), "null"), (dict(w_codes=4104), "aligned"), (dict(y_row_stride=7), "y_row_stride"),
                     (dict(out_features=-2), "rows")):
        assert call(**kw) == -1 and word in _message(lib), kw
    assert call(ws=None) == -4 and "needed" in _message(lib)
    assert call(ws_bytes=16) == -4
    assert call(ws=C.c_void_p(4097)) == -4 and "aligned" in _message(lib)
    assert call(rows=0, x=None) == 0 and call(out_features=0) == 0
    assert lib.nnb_mx4_linear(None, None, None, 0) == -1
    n = C.c_size_t()
    assert lib.nnb_mx4_linear_workspace_bytes(4, 64, 8, 0, None) == -1
    assert lib.nnb_mx4_linear_workspace_bytes(4, 64, 8, 0, C.byref(n)) == 0 and n.value >= 4 * (64 + 4)


def test_mx4_python_refusals():
    import torch
    from alphazero_amd import mx4
    from alphazero_amd._lib import NnbError
    codes, scales = torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8)
    w = mx4.MX4Tensor(codes, scales, (8, 100))
    for bad in ((codes, scales, (8, 300)), (codes, scales, (7, 100)), (codes.int(), scales, (8, 100)), (codes, scales, ()),
                (codes, scales, (8, 0)), (codes[:, ::2], scales, (8, 60))):
        with pytest.raises(ValueError):
            mx4.MX4Tensor(*bad)
    with pytest.raises(ValueError):
        mx4.quantize(torch.zeros(4, 64, dtype=torch.int32))
    with pytest.raises(ValueError):
        mx4.quantize(torch.zeros(4, 64, dtype=torch.float64))
    with pytest.raises(ValueError):
        mx4.quantize(torch.zeros(4, 0))
    with pytest.raises(ValueError):
        mx4.quantize(torch.tensor(1.0))
    x = torch.zeros(3, 100)
    with pytest.raises(NnbError):                                       # no CPU path
        mx4.quantize(x)
    with pytest.raises(NnbError):
        mx4.linear(x, w)
    with pytest.raises(NnbError):
        w.dequantize()
    for kw in (dict(x=torch.zeros(3, 99)), dict(bias=torch.zeros(7)), dict(x=torch.zeros(3, 100).double()),
               dict(weight=torch.zeros(8, 100))):
        with pytest.raises(ValueError):
            mx4.linear(**{**dict(x=x, weight=w), **kw})
    with pytest.raises(NnbError, match="backward"):
        mx4.linear(x.clone().requires_grad_(), w)
    with pytest.raises(NnbError, match="backward"):
        mx4.quantize(x.clone().requires_grad_())
