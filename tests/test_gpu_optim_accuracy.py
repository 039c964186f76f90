"""Orthogonalisation is as accurate as the formula computed in plain float32, on every path its size can take."""
import pytest

pytestmark = pytest.mark.gpu


def _formula(x, steps=5, abc=(3.4445, -4.7750, 2.0315)):
    """In x's own precision; every matrix of the batch has rows <= cols."""
    x = x / (x.norm(dim=(-2, -1), keepdim=True) + 1e-7)
    for _ in range(steps):
        g = x @ x.mT.contiguous()
        x = abc[0] * x + (abc[1] * g + abc[2] * (g @ g)) @ x
    return x


# one block; one launch per segment (64 and 128 rows); a launch per product on 64 x 64 tiles with two groups of waves and
# with one; on 128 x 128 tiles, one large matrix and a batch; a long side cut into parts
SHAPES = [(32, 128), (60, 190), (40, 4000), (100, 130), (2, 128, 2048), (200, 3000), (1024, 1100), (3, 777, 1501),
          (2450, 2600), (8, 900, 1000)]


@pytest.mark.parametrize("shape", SHAPES)
def test_error_within_three_times_plain_float32(shape):
    """Both forms round to 24 (22) bits and add in float32, in different orders; what their errors have in common is the
    growth in the directions of small singular values, which the plain form's error measures for this very matrix.  A
    factor of two for the 22 bits of the operands (2^-23 against 2^-24 per rounding), half as much again for the orders."""
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X (torch.cuda.is_available() is False)")
    from alphazero_amd import optim
    x = torch.randn(shape, generator=torch.Generator().manual_seed(shape[-1])).cuda()
    want = _formula(x.double())
    size = want.norm()
    ours, plain = ((y.double() - want).norm() / size for y in (optim.orthogonalize(x), _formula(x)))
    assert ours <= 3 * plain, (ours.item(), plain.item())
    turned = optim.orthogonalize(x.mT.contiguous()).mT
    assert (turned.double() - want).norm() / size <= 3 * plain
