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
