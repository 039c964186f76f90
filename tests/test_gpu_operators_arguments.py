"""The matrix operators on unusual but legal tensors: they see what torch sees."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X (torch.cuda.is_available() is False)")
    return torch


def test_negated_views_read_as_their_negative():
    """The imaginary part of a conjugate is a float32 tensor that shares memory with the un-negated numbers."""
    torch = _torch()
    from alphazero_amd import mx4, optim
    g = torch.Generator().manual_seed(1)
    draw = lambda *s: torch.randn(s, generator=g).cuda()
    # from complex numbers, and a contiguous one as torch may hand it on
    for negate in (lambda t: torch.complex(torch.zeros_like(t), t).conj().imag, torch._neg_view):
        x, w, b = draw(20, 70), draw(40, 70), draw(40)
        nx = negate(x)
        assert nx.is_neg()
        assert torch.equal(mx4.quantize(nx).dequantize(), -mx4.quantize(x).dequantize())
        weight = mx4.quantize(w)
        assert torch.equal(mx4.linear(nx, weight, bias=negate(b)), mx4.linear(-x, weight, bias=-b))
        assert torch.equal(mx4.linear(nx.view(4, 5, 70), weight), mx4.linear((-x).view(4, 5, 70), weight))
        assert torch.equal(optim.orthogonalize(nx), optim.orthogonalize(-x))
        assert torch.equal(optim.orthogonalize(x, out=x), optim.orthogonalize(-nx))
    m = draw(20, 70) * 1e-3
    x, w = draw(20, 70), draw(20, 70)
    want = optim.muon_update([w], [-x], [m], lr=0.1, inplace=False)
    assert all(torch.equal(a[0], c[0]) for a, c in zip(optim.muon_update([w], [torch._neg_view(x)], [m], lr=0.1, inplace=False), want))
    want = optim.muon_update([-w], [x], [-m], lr=0.1, inplace=False)
    got = optim.muon_update([torch._neg_view(w)], [x], [torch._neg_view(m)], lr=0.1, inplace=False)
    assert all(torch.equal(a[0], c[0]) for a, c in zip(got, want))
