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
