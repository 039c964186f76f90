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
        assert torch.equal(optim.orthogonalize(-nx), optim.orthogonalize(x))
    m = draw(20, 70) * 1e-3
    x, w = draw(20, 70), draw(20, 70)
    want = optim.muon_update([w], [-x], [m], lr=0.1, inplace=False)
    assert all(torch.equal(a[0], c[0]) for a, c in zip(optim.muon_update([w], [torch._neg_view(x)], [m], lr=0.1, inplace=False), want))
    want = optim.muon_update([-w], [x], [-m], lr=0.1, inplace=False)
    got = optim.muon_update([torch._neg_view(w)], [x], [torch._neg_view(m)], lr=0.1, inplace=False)
    assert all(torch.equal(a[0], c[0]) for a, c in zip(got, want))


def test_muon_in_a_graph_behind_one_eager_step():
    torch = _torch()
    from alphazero_amd import optim
    from alphazero_amd._lib import NnbError
    g = torch.Generator().manual_seed(2)
    start, grad = torch.randn(40, 90, generator=g).cuda(), torch.randn(40, 90, generator=g).cuda()
    eager, p = (torch.nn.Parameter(start.clone()) for _ in range(2))
    eager.grad, p.grad = grad.clone(), grad.clone()
    a, b = optim.Muon([eager], lr=0.1), optim.Muon([p], lr=0.1)
    with pytest.raises(NnbError, match="momentum"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            b.step()
    assert torch.equal(p, start)
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for k in range(4):
        for t in (eager, p):
            t.grad.copy_(grad * (k + 2))
        a.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(p, eager) and torch.equal(a.state[eager]["momentum"], b.state[p]["momentum"]), k
