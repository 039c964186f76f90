"""Self-play, training with Muon and the network's 4-bit evaluation, used together."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X (torch.cuda.is_available() is False)")
    return torch


@pytest.mark.parametrize("precision", ["mx4", "f32s"])
def test_play_train_play(precision):
    torch = _torch()
    from alphazero_amd.agent import initialize_agent
    from alphazero_amd.engine import Engine
    from alphazero_amd.selfplay import self_play_sample_tensors, train_network
    torch.manual_seed(0)
    agent = initialize_agent(use_gpu=True, num_simulations=24, load_model=False)
    agent.precision = precision
    samples = self_play_sample_tensors(agent, 6)
    before = {k: v.clone() for k, v in agent.model.state_dict().items()}
    losses = train_network(agent, *samples, epochs=2, batch_size=16)
    assert len(losses) == 2 and all(np.isfinite(losses))
    after = agent.model.state_dict()
    assert all(torch.isfinite(v).all() for v in after.values())
    assert all(not torch.equal(before[k], after[k]) for k in after)
    # the agent's engine evaluates the trained weights: as an engine that has never seen others
    planes = samples[0]
    eng, fresh = agent.engine(len(planes)), Engine(max_games=len(planes), max_sims=24, precision=precision)
    try:
        fresh.load_state_dict(after)
        for a, b in zip(eng.net_forward_planes(planes), fresh.net_forward_planes(planes)):
            assert torch.equal(a, b)
    finally:
        fresh.close()
    again = self_play_sample_tensors(agent, 6)
    assert len(again[0]) > 0 and torch.isfinite(again[1]).all()


def test_train_network_arguments_and_time_limit():
    torch = _torch()
    from alphazero_amd.agent import initialize_agent
    from alphazero_amd.selfplay import self_play_sample_tensors, train_network
    agent = initialize_agent(use_gpu=True, num_simulations=8, load_model=False)
    planes, probs, z = self_play_sample_tensors(agent, 2)
    assert train_network(agent, planes[:0], probs[:0], z[:0]) == []
    assert len(train_network(agent, planes, probs, z, epochs=50, time_limit=0.0)) == 1
    with pytest.raises(ValueError):
        train_network(agent, planes, probs[1:], z)
    with pytest.raises(ValueError):
        train_network(agent, planes, probs, z, batch_size=0)


def test_train_alphazero_plays_trains_and_saves(tmp_path, monkeypatch):
    torch = _torch()
    from alphazero_amd.agent import MODEL_PATH
    from alphazero_amd.selfplay import train_alphazero
    monkeypatch.chdir(tmp_path)
    agent = train_alphazero(time_limit=0.5, num_self_play_games=2, use_gpu=True, load_model=False)
    saved = torch.load(MODEL_PATH, map_location=agent.device, weights_only=True)
    assert all(torch.equal(saved[k], v) for k, v in agent.model.state_dict().items())
    with pytest.raises(FileNotFoundError):
        monkeypatch.chdir(tmp_path.parent)
        train_alphazero(time_limit=0.5, num_self_play_games=1, use_gpu=True, load_model=True)


def test_outputs_over_inputs_are_refused_and_seen_by_torch():
    torch = _torch()
    from alphazero_amd import mx4, optim
    x = torch.randn(12, 64, generator=torch.Generator().manual_seed(1)).cuda()
    weight = mx4.quantize(torch.randn(64, 64, generator=torch.Generator().manual_seed(2)).cuda())
    for out in (x, x[:, :], x.view(-1)[:768].view(12, 64)):
        with pytest.raises(ValueError, match="shares memory"):
            mx4.linear(x, weight, out=out)
    other = torch.zeros(13, 64, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        mx4.linear(x, weight, bias=other[11], out=other[:12])
    wide = torch.randn(12, 128, generator=torch.Generator().manual_seed(3)).cuda()
    before, version = wide.clone(), wide._version
    mx4.linear(wide[:, :64], weight, out=wide[:, 64:])
    assert wide._version > version and torch.equal(wide[:, :64], before[:, :64])
    assert torch.equal(wide[:, 64:], mx4.linear(before[:, :64], weight))
    with pytest.raises(ValueError, match="shares memory"):
        optim.orthogonalize(wide[:8], out=wide[4:])
    with pytest.raises(ValueError, match="shares memory"):
        optim.orthogonalize(wide[:, :12], out=wide[:, :12].t())
    square, version = wide[:, 64:], wide._version
    want = optim.orthogonalize(square.clone())
    optim.orthogonalize(square, out=square)
    assert torch.equal(square, want) and wide._version > version
    w, g, m = (torch.zeros(4, 8, device="cuda") for _ in range(3))
    flat = torch.zeros(60, device="cuda")
    for args in (([w, w], [g, g], [m, torch.zeros_like(m)]), ([w], [w], [m]), ([w], [m], [m]),
                 ([flat[:32].view(4, 8), flat[28:].view(4, 8)], [g, g], [m, torch.zeros_like(m)])):
        with pytest.raises(ValueError, match="shares memory"):
            optim.muon_update(*args, lr=0.1)
    optim.muon_update([w, torch.ones_like(w)], [g, g], [m, torch.zeros_like(m)], lr=0.1)      # one gradient twice is no matter
