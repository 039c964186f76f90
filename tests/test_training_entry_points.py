"""What train_alphazero, train_network and AlphaZeroAgent.perform_training do around the games and the kernels, without a GPU:
the games come from a stand-in."""
import pytest
import torch


@pytest.fixture
def played(monkeypatch):
    """Any game played is noted here instead."""
    from alphazero_amd.agent import AlphaZeroAgent
    calls = []

    def engine(self, *args, **kwargs):
        calls.append(args)
        raise AssertionError("a game was about to be played")
    monkeypatch.setattr(AlphaZeroAgent, "engine", engine)
    return calls


def test_training_on_the_cpu_is_refused_before_a_game_is_played(played):
    from alphazero_amd.agent import initialize_agent
    from alphazero_amd.selfplay import train_alphazero, train_network
    with pytest.raises(RuntimeError, match="GPU"):
        train_alphazero(time_limit=1, num_self_play_games=2, use_gpu=False, load_model=False)
    agent = initialize_agent(load_model=False)
    with pytest.raises(RuntimeError, match="GPU"):
        agent.perform_training()
    with pytest.raises(RuntimeError, match="GPU"):
        train_network(agent, torch.zeros(4, 2, 6, 7), torch.zeros(4, 7), torch.zeros(4))
    assert not played


@pytest.fixture
def stand_ins(monkeypatch, tmp_path):
    """Self-play and the fit replaced: notes who plays, who is fitted to what, and where the result is saved."""
    from alphazero_amd import selfplay
    notes = []
    monkeypatch.chdir(tmp_path)
    monkeypatch.setattr(selfplay, "_check_trainable", lambda agent: None)
    monkeypatch.setattr(selfplay, "_play_for_training", lambda agent, n: notes.append(("play", agent, n)) or ("planes", "probs", "z"))
    monkeypatch.setattr(selfplay, "train_network",
                        lambda agent, *samples, **kw: notes.append(("fit", agent, samples, kw["time_limit"])) or [])
    return notes


def test_perform_training_trains_the_agent_itself(stand_ins):
    from alphazero_amd.agent import MODEL_PATH, initialize_agent
    agent = initialize_agent(load_model=False)
    with torch.no_grad():
        agent.model.value_head.bias.fill_(3.0)
    agent.perform_training()
    assert stand_ins == [("play", agent, 1000), ("fit", agent, ("planes", "probs", "z"), 3600)]
    assert torch.load(MODEL_PATH, weights_only=True)["value_head.bias"].item() == 3.0


def test_train_alphazero_trains_the_agent_it_returns(stand_ins):
    from alphazero_amd.selfplay import train_alphazero
    agent = train_alphazero(7.5, num_self_play_games=3, use_gpu=False, load_model=False)
    assert stand_ins == [("play", agent, 3), ("fit", agent, ("planes", "probs", "z"), 7.5)]
    assert (agent.num_simulations, agent.c_puct) == (800, 1.4)


class _Engine:
    """Two finished games, as an engine returns them."""
    def __init__(self):
        import numpy as np
        from alphazero_amd.engine import TRAJECTORY_DTYPE
        self.records = np.zeros(2, dtype=TRAJECTORY_DTYPE)
        for r, length, result in zip(self.records, (7, 8), (1, -1)):
            r["length"], r["result"] = length, result
            r["plies"]["player"][:length] = [1 + i % 2 for i in range(length)]
        self.rounds = 0

    def params(self, *args, **kwargs):
        return None

    def selfplay_round(self, n, params, **kwargs):
        import numpy as np
        self.rounds += 1
        return torch.from_numpy(self.records.view(np.uint8).reshape(2, -1).copy()), {"games": 2, "plies": 15, "sims": 1}

    def trajectory_samples(self, traj):
        return traj, None, None


def test_training_fills_the_agents_memory_as_self_play_does(monkeypatch):
    from alphazero_amd import selfplay
    from alphazero_amd.agent import AlphaZeroAgent, initialize_agent
    engine, agent, other = _Engine(), initialize_agent(load_model=False), initialize_agent(load_model=False)
    monkeypatch.setattr(AlphaZeroAgent, "engine", lambda self, *a, **k: engine)
    traj, _, _ = selfplay._play_for_training(agent, 2)
    assert engine.rounds == 1 and traj.shape[0] == 2                  # one set of games for both
    selfplay.self_play(other, 2)
    assert len(agent.memory) == 2 and [m[2] for m in agent.memory] == [m[2] for m in other.memory] == [1, -1]
    for a, b in zip(agent.memory, other.memory):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_training_in_several_processes_is_refused(stand_ins, monkeypatch):
    """Each would play the same games, train by itself and write the same file."""
    import torch.distributed as dist
    from alphazero_amd.agent import initialize_agent
    from alphazero_amd.selfplay import train_alphazero
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_world_size", lambda group=None: 2)
    with pytest.raises(RuntimeError, match="process"):
        train_alphazero(1.0, num_self_play_games=2, use_gpu=False, load_model=False)
    with pytest.raises(RuntimeError, match="process"):
        initialize_agent(load_model=False).perform_training()
    assert not stand_ins
    monkeypatch.setattr(dist, "get_world_size", lambda group=None: 1)
    train_alphazero(1.0, num_self_play_games=2, use_gpu=False, load_model=False)
    assert len(stand_ins) == 2
