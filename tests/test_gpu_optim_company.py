"""The optimiser step treats a matrix as precisely beside others as by itself."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X (torch.cuda.is_available() is False)")
    return torch


def _orthogonalized(xs):
    """What muon_update subtracts: weights and momenta of zero, lr = 1, no momentum."""
    import torch
    from alphazero_amd import optim
    w, _ = optim.muon_update([torch.zeros_like(x) for x in xs], xs, [torch.zeros_like(x) for x in xs], lr=1.0, momentum=0.0,
                             nesterov=False, inplace=False)
    return [-y / math.sqrt(max(1.0, x.shape[0] / x.shape[1])) for y, x in zip(w, xs)]


def test_products_of_lo_halves_go_by_the_matrix_itself():
    """They are taken for squares of up to 512 rows.  With 200 x 900 alone and beside 600 x 900 the same tiles multiply, so
    that not a bit may differ."""
    torch = _torch()
    g = torch.Generator().manual_seed(1)
    small, large = torch.randn(200, 900, generator=g).cuda(), torch.randn(600, 900, generator=g).cuda()
    alone, beside = _orthogonalized([small]), _orthogonalized([small, large])
    assert torch.equal(alone[0], beside[0])
    assert torch.equal(_orthogonalized([large])[0], beside[1])


def _formula(x, steps=5, abc=(3.4445, -4.7750, 2.0315)):
    """In x's own precision."""
    tall = x.shape[0] > x.shape[1]
    x = x.T.contiguous() if tall else x
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        g = x @ x.T.contiguous()
        x = abc[0] * x + (abc[1] * g + abc[2] * (g @ g)) @ x
    return x.T if tall else x


def _matrix(kind, rows, cols, seed):
    """Normal numbers; rows and columns of different sizes, as gradients have; singular values over three decades."""
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if kind == "gradient":
        x = x * torch.exp(0.5 * torch.randn(rows, 1, generator=g)) * torch.exp(0.5 * torch.randn(1, cols, generator=g)) * 1e-3
    if kind == "decaying":
        u, _, v = torch.linalg.svd(x.double(), full_matrices=False)
        x = (u * 10.0 ** torch.linspace(0, -3, min(rows, cols), dtype=torch.float64) @ v).float()
    return x.cuda()


# up to 128 rows, beside matrices of more than 128, of more than 512, and the network's own convolutions
LISTS = {"large": [(128, 2048), (7, 1024), (600, 900)], "middle": [(100, 130), (60, 1000), (515, 129), (300, 211)],
         "many": [(65, 130), (128, 128), (200, 3000), (130, 140), (512, 512), (640, 700)]}


@pytest.mark.parametrize("kind", ["normal", "gradient", "decaying"])
@pytest.mark.parametrize("shapes", LISTS.values(), ids=LISTS)
def test_precision_does_not_depend_on_the_other_matrices(shapes, kind):
    """Each matrix of a list: at most three times the plain float32 form's error, and three times its own error alone, which
    is no more than three times the plain form's either (see test_gpu_optim_accuracy for these two).  What
    rounds is the same in both cases, but for the terms with a diagonal, 24 bits of the other factor alone and 22 + 1 (a
    sign) beside others, a factor of two; half as much again for sums in another order."""
    torch = _torch()
    xs = [_matrix(kind, r, c, i + 1) for i, (r, c) in enumerate(shapes)]
    beside = _orthogonalized(xs)
    for x, y in zip(xs, beside):
        want = _formula(x.double())
        error = lambda t: ((t.double() - want).norm() / want.norm()).item()
        alone, plain = error(_orthogonalized([x])[0]), error(_formula(x))
        assert alone <= 3 * plain and error(y) <= 3 * plain and error(y) <= 3 * alone, (tuple(x.shape), error(y), alone, plain)


@pytest.mark.parametrize("kind", ["normal", "gradient", "decaying"])
@pytest.mark.parametrize("shapes", [[(33, 70), (128, 32), (128, 2048), (600, 900)], [(64, 64), (33, 33), (515, 129), (300, 211)],
                                    [(33, 33)] * 3 + [(65, 130), (640, 700), (190, 60)]], ids=["large", "middle", "many"])
def test_small_matrices_take_their_own_way(shapes, kind):
    """Up to 64 x 192 alone a matrix is formed afresh for every step, and so it has to be beside others: the same bounds."""
    test_precision_does_not_depend_on_the_other_matrices(shapes, kind)


@pytest.mark.parametrize("rows,cols,batch", [(65, 66, 2000), (4, 5, 20000)])
def test_large_batches(rows, cols, batch):
    """2000 matrices of 65 x 66 need more workspace than one group of launches is given; many small ones need none."""
    torch = _torch()
    import ctypes
    from alphazero_amd import _lib, optim
    n = ctypes.c_size_t()
    _lib.check(_lib.load().nnb_orthogonalize_workspace_bytes(batch, rows, cols, ctypes.byref(n)), "bytes")
    one = ctypes.c_size_t()
    _lib.check(_lib.load().nnb_orthogonalize_workspace_bytes(1, rows, cols, ctypes.byref(one)), "bytes")
    assert n.value < batch * one.value
    x = torch.randn(batch, rows, cols, generator=torch.Generator().manual_seed(rows)).cuda()
    got = optim.orthogonalize(x).double()

    def formula(x):
        x = x / (x.norm(dim=(1, 2), keepdim=True) + 1e-7)
        for _ in range(5):
            g = x @ x.mT.contiguous()
            x = 3.4445 * x + (-4.7750 * g + 2.0315 * (g @ g)) @ x
        return x
    want = formula(x.double())
    error = lambda t: (t - want).norm(dim=(1, 2)) / want.norm(dim=(1, 2))
    ours, plain = error(got), error(formula(x).double())
    assert ours.pow(2).mean().sqrt() <= 3 * plain.pow(2).mean().sqrt()
    # one matrix's error goes by its smallest singular values, by this bound of the worst (see test_gpu_optim.FAITHFUL)
    assert ours.max() <= 2 * 2.0 ** -20 * 4.7750 * 3.4445 ** 3


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 7])
def test_step_counts_of_mixed_lists(steps, dtype):
    """A segment of one step ends with the product that another one begins with: its Q is whole at once.  The bound is that of
    test_gpu_optim (FAITHFUL), for the step's move from zero weights, and one rounding to the type."""
    torch = _torch()
    from alphazero_amd import optim
    half_step = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}[dtype]
    xs = [_matrix("gradient", r, c, i + 3).to(getattr(torch, dtype))
          for i, (r, c) in enumerate([(33, 70), (120, 250), (64, 400), (1, 300), (200, 300), (530, 600), (1, 1)])]
    w, _ = optim.muon_update([torch.zeros_like(x) for x in xs], xs, [torch.zeros(x.shape, device="cuda") for x in xs], lr=1.0,
                             momentum=0.0, nesterov=False, steps=steps, inplace=False)
    for x, y in zip(xs, w):
        want = -_formula(x.double(), steps) * math.sqrt(max(1.0, x.shape[0] / x.shape[1]))
        assert (y.double() - want).norm() <= (2 * 2.0 ** -20 * 4.7750 * 3.4445 ** 3 + half_step) * want.norm(), tuple(x.shape)


def test_zero_nan_and_infinity_beside_other_matrices():
    torch = _torch()
    shapes = [(40, 60), (100, 130), (1, 300), (2, 500), (150, 70), (600, 700)]
    xs = [_matrix("normal", r, c, i + 1) for i, (r, c) in enumerate(shapes)]
    want = _orthogonalized(xs)
    for i in range(len(shapes)):
        for value in (0.0, float("nan"), float("inf")):
            changed = [x.clone() for x in xs]
            if value == 0.0:
                changed[i].zero_()
            else:
                changed[i][-1, shapes[i][1] // 2] = value
            got = _orthogonalized(changed)
            assert not got[i].any() if value == 0.0 else got[i].isnan().all(), (i, value)
            assert all(torch.equal(a, b) for k, (a, b) in enumerate(zip(got, want)) if k != i), (i, value)
