"""Arguments that the matrix operators have to refuse or to read with care, checked without a GPU: what is refused is refused
before the tensors' device matters, what is accepted gets as far as that."""
import pytest


def test_muon_update_sees_memory_shared_inside_a_longer_gradient():
    """Ranges sorted by their start: the one in between ends before the weight begins, the first does not."""
    import torch
    from alphazero_amd import optim
    from alphazero_amd._lib import NnbError
    flat, z = torch.zeros(1000), torch.zeros
    outer, inner, weight = flat[:900].view(30, 30), flat[10:14].view(2, 2), flat[500:504].view(2, 2)
    with pytest.raises(ValueError, match="shares memory"):
        optim.muon_update([z(30, 30), weight], [outer, inner], [z(30, 30), z(2, 2)], lr=0.1)
    # a written range that holds a gradient two places on, and two written ranges around a gradient of their own
    with pytest.raises(ValueError, match="shares memory"):
        optim.muon_update([outer, z(2, 2), z(2, 2)], [z(30, 30), z(2, 2), inner], [z(30, 30), z(2, 2), z(2, 2)], lr=0.1)
    with pytest.raises(ValueError, match="shares memory"):
        optim.muon_update([outer, weight], [z(30, 30), z(2, 2)], [z(30, 30), z(2, 2)], lr=0.1)
    # gradients may share memory with each other, and neighbours may touch: only the device is wrong then
    with pytest.raises(NnbError):
        optim.muon_update([flat[900:904].view(2, 2), z(30, 30)], [inner, outer], [z(2, 2), z(30, 30)], lr=0.1)


def _negated(t):
    """-t as torch makes it for the imaginary part of a conjugate: t's own memory and a mark."""
    import torch
    view = torch.complex(torch.zeros_like(t), t).conj().imag
    assert view.is_neg() and torch.equal(view, -t)
    return view


def test_negated_views_are_not_written_to():
    import torch
    from alphazero_amd import mx4, optim
    weight = mx4.MX4Tensor(torch.zeros(1, 1, 4096, dtype=torch.uint8), torch.zeros(1, 1, 256, dtype=torch.uint8), (8, 64))
    x = torch.ones(3, 64)
    with pytest.raises(ValueError, match="negated"):
        mx4.linear(x, weight, out=torch._neg_view(torch.zeros(3, 8)))
    with pytest.raises(ValueError, match="negated"):
        optim.orthogonalize(x, out=_negated(x))
    with pytest.raises(ValueError, match="negated"):
        optim.orthogonalize(_negated(x), out=_negated(x))
    z = torch.zeros
    for which in (0, 2):
        args = [[z(4, 8)], [z(4, 8)], [z(4, 8)]]
        args[which][0] = torch._neg_view(z(4, 8))
        with pytest.raises(ValueError, match="negated"):
            optim.muon_update(*args, lr=0.1)


def test_forward_mode_tangents_are_refused():
    """The kernels would return a result without a tangent, which reads as a derivative of zero."""
    import torch
    import torch.autograd.forward_ad as fwd
    from alphazero_amd import mx4, optim
    from alphazero_amd._lib import NnbError
    weight = mx4.MX4Tensor(torch.zeros(1, 1, 4096, dtype=torch.uint8), torch.zeros(1, 1, 256, dtype=torch.uint8), (8, 64))
    x, z = torch.ones(8, 64), torch.zeros
    with fwd.dual_level():
        dual = fwd.make_dual(x, x)
        for guard in (torch.enable_grad, torch.no_grad):              # neither switches tangents on or off
            with guard():
                for call in (lambda: mx4.quantize(dual), lambda: mx4.linear(dual, weight),
                             lambda: mx4.linear(x, weight, bias=fwd.make_dual(z(8), z(8))), lambda: optim.orthogonalize(dual),
                             lambda: mx4.linear(x, weight, out=fwd.make_dual(z(8, 8), z(8, 8))),
                             lambda: optim.orthogonalize(x, out=fwd.make_dual(z(8, 64), x)),
                             lambda: optim.muon_update([x.clone()], [dual], [z(8, 64)], lr=0.1),
                             lambda: optim.muon_update([fwd.make_dual(x.clone(), x)], [x], [z(8, 64)], lr=0.1, inplace=False),
                             lambda: optim.muon_update([x.clone()], [x], [fwd.make_dual(z(8, 64), x)], lr=0.1)):
                    with pytest.raises(NnbError, match="forward-mode"):
                        call()
        for call in (lambda: mx4.quantize(x), lambda: optim.muon_update([x.clone()], [x], [z(8, 64)], lr=0.1)):
            with pytest.raises(NnbError, match="no CPU path"):        # a plain tensor under a dual level is as good as any
                call()


def test_orthogonalize_refuses_an_out_that_overlaps_itself():
    import torch
    from alphazero_amd import optim
    from alphazero_amd._lib import NnbError
    x, flat = torch.zeros(6, 20), torch.zeros(400)
    for out in (flat[:25].unfold(0, 20, 1), flat.as_strided((6, 20), (19, 1)), flat.as_strided((6, 20), (3, 4)),
                flat.as_strided((6, 20), (0, 1))):
        with pytest.raises(ValueError, match="share memory"):
            optim.orthogonalize(x, out=out)
    windows = flat[:25].unfold(0, 20, 1)                              # reading overlapping rows is fine, writing over them is not
    with pytest.raises(ValueError, match="share memory"):
        optim.orthogonalize(windows, out=windows)
    with pytest.raises(ValueError, match="share memory"):
        optim.orthogonalize(x.expand(3, 6, 20), out=flat.as_strided((3, 6, 20), (119, 20, 1)))
    for out in (flat.as_strided((6, 20), (20, 1)), flat.as_strided((6, 20), (1, 6)), flat.as_strided((6, 20), (41, 2)),
                flat[1:].as_strided((6, 20), (1, 7))):
        with pytest.raises(NnbError, match="no CPU path"):
            optim.orthogonalize(x, out=out)
    with pytest.raises(NnbError, match="no CPU path"):                # a stride of a dimension of one says nothing
        optim.orthogonalize(x[:1], out=flat.as_strided((1, 20), (1, 1)))


def test_muon_on_the_cpu_says_that_it_has_no_path_there():
    import torch
    from alphazero_amd import optim
    from alphazero_amd._lib import NnbError
    p = torch.nn.Parameter(torch.randn(4, 8))
    p.grad = torch.ones(4, 8)
    with pytest.raises(NnbError, match="no CPU path"):
        optim.Muon([p], lr=0.1).step()


def test_mx4_linear_refuses_more_features_than_a_grid_holds():
    """A launch has less than 2^32 threads, 512 for every 16 features."""
    import ctypes as C
    from alphazero_amd import _lib
    lib, n, most = _lib.load(), C.c_size_t(), 2 ** 27 - 16
    for rows in (0, 1, 40):
        assert lib.nnb_mx4_linear_workspace_bytes(rows, 32, most, 0, C.byref(n)) == 0
        for features in (most + 1, 2 ** 27, 2 ** 31 - 1):
            assert lib.nnb_mx4_linear_workspace_bytes(rows, 32, features, 0, C.byref(n)) == -1
            assert "features" in lib.nnb_last_error().decode()
            a = _lib.Mx4LinearArgs(rows=rows, cols=32, out_features=features, x=4096, x_row_stride=32, x_col_stride=1,
                                   w_codes=4096, w_scales=4096, y=4096, y_row_stride=features)
            assert lib.nnb_mx4_linear(None, C.byref(a), C.c_void_p(4096), 1 << 30) == -1


def test_matrices_in_one_blocks_lds_need_no_workspace_of_their_own():
    import ctypes as C
    from alphazero_amd import _lib
    lib, n = _lib.load(), C.c_size_t()

    def muon(*shapes):
        items = (_lib.MuonMatrix * len(shapes))(*[_lib.MuonMatrix(rows=r, cols=c) for r, c in shapes])
        assert lib.nnb_muon_workspace_bytes(len(shapes), items, C.byref(n)) == 0
        return n.value
    for batch, rows, cols in ((1, 1, 1), (1 << 20, 64, 64), ((1 << 31) - 1, 64, 192), (7, 192, 64)):
        assert lib.nnb_orthogonalize_workspace_bytes(batch, rows, cols, C.byref(n)) == 0 and n.value == 256, (rows, cols)
    assert muon((64, 64)) == muon(*[(3, 5)] * 100) == 256
    assert muon() == muon((0, 5), (7, 0)) == 0
    large = muon((200, 300))
    assert large > 1 << 20 and muon((64, 64), (200, 300), (192, 64)) == large and muon((65, 193), (200, 300)) > large


ROWS, ONE_PER_CU, TWO_PER_CU, LARGE = range(4)


# measured either side of where one form becomes faster than another (profiles/mx4_forms.txt)
@pytest.mark.parametrize("rows,cols,out,y_type,form", [
    (1, 11520, 1024, 0, ROWS), (512, 11520, 1024, 2, ROWS), (2048, 11520, 1024, 2, ONE_PER_CU), (4096, 11520, 1024, 0, ONE_PER_CU),
    (8192, 11520, 1024, 2, TWO_PER_CU), (64, 8192, 8192, 2, ROWS), (256, 8192, 8192, 2, ONE_PER_CU), (1024, 8192, 8192, 2, TWO_PER_CU),
    (2048, 8192, 8192, 2, LARGE), (8192, 8192, 8192, 2, LARGE), (17, 1024, 8192, 2, ROWS), (64, 1024, 8192, 0, ROWS),
    (512, 1024, 8192, 2, ONE_PER_CU), (2048, 1024, 8192, 2, TWO_PER_CU), (64, 256, 2048, 2, ROWS), (512, 256, 2048, 2, ONE_PER_CU),
    (8192, 256, 2048, 2, TWO_PER_CU), (2048, 4096, 4096, 2, TWO_PER_CU), (4096, 4096, 4096, 2, LARGE), (4096, 4096, 4096, 0, LARGE),
    (512, 1024, 1024, 0, ROWS), (2048, 1024, 1024, 2, ONE_PER_CU), (8192, 256, 8192, 2, TWO_PER_CU), (1024, 16384, 300, 2, ROWS),
    (8192, 16384, 300, 2, ONE_PER_CU), (86, 102, 489, 0, ROWS), (1957, 193, 213, 0, ROWS), (5084, 9483, 171, 0, ONE_PER_CU)])
def test_mx4_linear_takes_the_form_that_measured_fastest(rows, cols, out, y_type, form):
    from alphazero_amd import _lib
    assert _lib.load().nnb_debug_mx4_form(rows, cols, out, y_type) == form


def test_mx4_form_refuses_what_the_product_refuses():
    from alphazero_amd import _lib
    lib = _lib.load()
    for args in ((-1, 64, 8, 0), (4, 0, 8, 0), (4, 64, 2 ** 27, 0), (4, 64, 8, 3)):
        assert lib.nnb_debug_mx4_form(*args) == -1
