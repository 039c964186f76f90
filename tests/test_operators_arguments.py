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
