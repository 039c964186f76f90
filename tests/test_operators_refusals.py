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
    assert call(rows=40, ws=None) == -4 and "needed" in _message(lib)
    assert call(rows=40, ws_bytes=16) == -4
    assert call(rows=40, ws=C.c_void_p(4097)) == -4 and "aligned" in _message(lib)
    assert call(rows=0, x=None) == 0 and call(out_features=0) == 0
    assert lib.nnb_mx4_linear(None, None, None, 0) == -1
    n = C.c_size_t()
    assert lib.nnb_mx4_linear_workspace_bytes(4, 64, 8, 0, None) == -1
    assert lib.nnb_mx4_linear_workspace_bytes(4, 64, 8, 0, C.byref(n)) == 0 and n.value == 0
    assert lib.nnb_mx4_linear_workspace_bytes(40, 11520, 8, 0, C.byref(n)) == 0 and n.value >= 40 * (5760 + 360)


def test_mx4_python_refusals():
    import torch
    from alphazero_amd import mx4
    from alphazero_amd._lib import NnbError
    codes, scales = torch.zeros(1, 1, 4096, dtype=torch.uint8), torch.zeros(1, 1, 256, dtype=torch.uint8)
    w = mx4.MX4Tensor(codes, scales, (8, 100))
    for bad in ((codes, scales, (8, 300)), (codes, scales, (33, 100)), (codes.int(), scales, (8, 100)), (codes, scales, ()),
                (codes, scales, (8, 0)), (codes.expand(2, 1, 4096), scales.expand(2, 1, 256), (40, 100)), (codes, scales[:, :, :128], (8, 100))):
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


def test_optimiser_structs_match_the_header(tmp_path):
    import os
    import subprocess
    from alphazero_amd import _lib
    from conftest import ROOT
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "nnb.h"\nint main(void){printf("%zu %zu %zu\\n",sizeof(nnb_newton_schulz),'
                   "sizeof(nnb_muon_matrix),sizeof(nnb_muon_params));return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    sizes = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert sizes == [C.sizeof(_lib.NewtonSchulz), C.sizeof(_lib.MuonMatrix), C.sizeof(_lib.MuonParams)]


def _ns(steps=5, abc=(3.4445, -4.7750, 2.0315), eps=1e-7):
    from alphazero_amd._lib import NewtonSchulz
    ns = NewtonSchulz(steps=steps, eps=eps)
    for i in range(16):
        for j in range(3):
            ns.coefficients[i][j] = abc[j]
    return ns


def test_orthogonalize_refuses_bad_arguments(lib):
    p, s = C.c_void_p(4096), (C.c_int64 * 3)(0, 64, 1)
    def call(t=0, batch=1, rows=32, cols=64, x=p, xs=s, out=p, os_=s, ns=None, ws=p, nbytes=1 << 30):
        ns = _ns() if ns is None else ns
        return lib.nnb_orthogonalize(None, t, batch, rows, cols, x, xs, out, os_, C.byref(ns), ws, nbytes)
    for kw, word in ((dict(t=4), "dtype"), (dict(batch=-1), "batch"), (dict(rows=-1), "matrix"), (dict(rows=20000, cols=20000), "16384"),
                     (dict(rows=1 << 16, cols=1 << 15), "16384"), (dict(cols=1 << 31), "2^31"), (dict(x=None), "null"),
                     (dict(out=None), "null"), (dict(xs=None), "null"), (dict(os_=None), "null"), (dict(ns=_ns(steps=0)), "steps"),
                     (dict(ns=_ns(steps=17)), "steps"), (dict(ns=_ns(eps=-1.0)), "eps"), (dict(ns=_ns(eps=float("nan"))), "eps"),
                     (dict(ns=_ns(abc=(float("inf"), 0.0, 0.0))), "finite"), (dict(ns=_ns(abc=(30.0, 0.0, 5.0))), "grow")):
        assert call(**kw) == -1 and word in _message(lib), kw
    assert call(ws=None) == -4 and call(nbytes=100) == -4 and call(ws=C.c_void_p(4100)) == -4
    assert call(batch=0, x=None) == 0 and call(rows=0) == 0 and call(cols=0) == 0
    assert lib.nnb_orthogonalize(None, 0, 1, 4, 4, p, s, p, s, None, p, 1 << 30) == -1
    n = C.c_size_t()
    assert lib.nnb_orthogonalize_workspace_bytes(1, 4, 4, None) == -1
    # a large batch is worked off in parts: its workspace stays bounded
    assert lib.nnb_orthogonalize_workspace_bytes(1 << 20, 64, 64, C.byref(n)) == 0 and 0 < n.value <= 1 << 30


def test_muon_step_refuses_bad_arguments(lib):
    from alphazero_amd._lib import MuonMatrix, MuonParams
    p = C.c_void_p(4096)
    def call(t=0, count=1, ws=p, nbytes=1 << 30, lr=0.1, momentum=0.9, wd=0.0, ns=None, **kw):
        items = (MuonMatrix * 2)()
        for it in items:
            for k, v in {**dict(weight=4096, grad=4096, momentum=4096, weight_out=4096, momentum_out=4096, rows=4, cols=8), **kw}.items():
                setattr(it, k, v)
        params = MuonParams(lr=lr, momentum=momentum, weight_decay=wd, nesterov=1, ns=_ns() if ns is None else ns)
        return lib.nnb_muon_step(None, t, count, items, C.byref(params), ws, nbytes)
    nan = float("nan")
    for kw, word in ((dict(t=-2), "dtype"), (dict(count=-1), "count"), (dict(lr=nan), "finite"), (dict(momentum=nan), "finite"),
                     (dict(wd=nan), "finite"), (dict(weight=None), "null"), (dict(grad=None), "null"), (dict(momentum_out=None), "null"),
                     (dict(rows=-3), "matrix"), (dict(ns=_ns(steps=40)), "steps")):
        assert call(**kw) == -1 and word in _message(lib), kw
    assert call(ws=None) == -4
    assert call(count=0, ws=None) == 0
    assert call(rows=0, ws=None, weight=None) == 0
    assert lib.nnb_muon_step(None, 0, 1, None, C.byref(MuonParams(ns=_ns())), p, 1) == -1
    assert lib.nnb_muon_step(None, 0, 1, None, None, p, 1) == -1


def test_optimiser_python_refusals():
    import torch
    from alphazero_amd import optim
    from alphazero_amd._lib import NnbError
    x = torch.randn(8, 9)
    with pytest.raises(NnbError):                                       # no CPU path
        optim.orthogonalize(x)
    for bad in (x[0], x.double(), x.int()):
        with pytest.raises(ValueError):
            optim.orthogonalize(bad)
    for kw in (dict(steps=0), dict(steps=17), dict(coefficients=(1.0, 2.0)), dict(coefficients=[(1, 0, 0)] * 4), dict(out=x.half()),
               dict(out=torch.zeros(9, 8))):
        with pytest.raises(ValueError):
            optim.orthogonalize(x, **kw)
    with pytest.raises(NnbError, match="backward"):
        optim.orthogonalize(x.clone().requires_grad_())
    w, g, m = x.clone(), x.clone(), x.clone()
    for args in (([w], [g], []), ([w], [g[:4]], [m]), ([w], [g.half()], [m]), ([w], [g], [m.half()]), ([w.double()], [g.double()], [m]),
                 ([w, w], [g, g], [m, m.clone()])):
        with pytest.raises(ValueError):
            optim.muon_update(*args, lr=0.1)
    with pytest.raises(NnbError):
        optim.muon_update([w], [g], [m], lr=0.1)
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(steps=0)):
        with pytest.raises(ValueError):
            optim.Muon([torch.nn.Parameter(x)], **kw)
    with pytest.raises(ValueError):
        optim.Muon([torch.nn.Parameter(x[0])])
    with pytest.raises(ValueError):
        optim.Muon([torch.nn.Parameter(x.t())])


def test_which_tensors_share_memory():
    import torch
    from alphazero_amd._tensors import share_memory
    buf = torch.zeros(8, 100)
    assert share_memory(buf, buf) and share_memory(buf[2:5], buf[4:]) and share_memory(buf[0], buf[:, 0])
    assert not share_memory(buf[:4], buf[4:]) and not share_memory(buf, torch.zeros(8, 100)) and not share_memory(buf[:0], buf)
    assert not share_memory(buf[:, :40], buf[:, 40:]) and not share_memory(buf[:, 40:], buf[:, :40])
    assert share_memory(buf[:, :41], buf[:, 40:]) and share_memory(buf[:, 40:], buf[:, :41])
    assert share_memory(buf[:, 60:], buf.view(-1)[90:].unfold(0, 20, 100))          # the second wraps around the row's end
    assert not share_memory(buf[:, 20:40], buf[1:, :20]) and not share_memory(buf[1:, :20], buf[:, 20:40])
    half = torch.zeros(8, 100, dtype=torch.float16)
    assert not share_memory(half[:, :50], half[:, 50:]) and share_memory(half[::2, :60], half[1:, 50:])


def test_matrices_near_the_limit_of_indices(lib):
    n = C.c_size_t()
    most = 2 ** 31 - 64
    for rows, cols in ((1, most + 1), (most + 63, 1), (7, 306783378), (16385, 16385)):
        assert lib.nnb_orthogonalize_workspace_bytes(1, rows, cols, C.byref(n)) == -1 and "2^31" in _message(lib), (rows, cols)
    for rows, cols in ((1, most), (most, 1), (16384, 131071)):
        assert lib.nnb_orthogonalize_workspace_bytes(1, rows, cols, C.byref(n)) == 0 and n.value > 12 * rows * cols, (rows, cols)
