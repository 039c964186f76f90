"""Engine(precision="mx4"): the policy-value network with its linear layer on 4-bit floats.

The layer is checked against float64 sums of the rounded operands: the activations it read (nnb_debug_activations
returns the halves exactly) and the weights, both rounded by mx4.quantize, whose own tests compare it with the
definition value by value.  The convolutions are those of precision="f16" bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rp():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X (torch.cuda.is_available() is False)")
    from oracle import ref_port
    return ref_port


def _positions(eng, n, seed):
    from alphazero_amd.selfplay import random_openings
    sb, sp = random_openings(eng, n, 6, seed=seed)
    return np.where(sp[:, None] == 1, sb, sb[:, ::-1]).astype(np.uint64), eng.game_ops(sb)[1]


@pytest.mark.parametrize("max_games,n", [(1, 1), (40, 5), (40, 40), (300, 299), (1500, 1500), (1500, 3)])
def test_forward_against_the_rounded_layer(rp, max_games, n):
    import torch
    from alphazero_amd import mx4
    from alphazero_amd.engine import Engine
    sd = rp.seeded_state_dict(0)
    eng, half = Engine(max_games=max_games, max_sims=2, precision="mx4"), Engine(max_games=max_games, max_sims=2, precision="f16")
    try:
        eng.load_state_dict(sd)
        half.load_state_dict(sd)
        side, legal = _positions(eng, n, seed=3)
        logp, value, priors = eng.net_forward(side, legal)
        half.net_forward(side, legal)
        a3 = eng.activations(3, n)
        assert torch.equal(a3, half.activations(3, n)) and torch.equal(eng.activations(2, n), half.activations(2, n))
        hidden = eng.activations(4, n).double().cpu()
    finally:
        eng.close()
        half.close()
    rows = a3.reshape(n, 11520)                                       # cell by cell, 128 channels each
    weight = sd["fc_layers.0.weight"].reshape(1024, 128, 90).permute(0, 2, 1).reshape(1024, 11520).contiguous().cuda()
    xq, wq = mx4.quantize(rows).dequantize().double().cpu(), mx4.quantize(weight).dequantize().double().cpu()
    sums, size = xq @ wq.T, xq.abs() @ wq.abs().T
    want = torch.relu(sums + sd["fc_layers.0.bias"].double())
    # the products are exact; 180 matrix instructions of 64 (or 90 of 128 in eight parts, then those) add in float32,
    # each off by at most 2^-23 of what they hold, then the bias and the rounding
    assert ((hidden - want).abs() <= 200 * 2.0 ** -23 * size + 2.0 ** -24 * want).all()
    # heads: 1024 fused steps in float32, half a step of the absolute sum each; then a logarithm of seven exponentials
    # (it passes its arguments' errors on at most twice) or a hyperbolic tangent, good to a few steps of values below 16
    heads = torch.cat([sd["policy_head.weight"], sd["value_head.weight"]]).double()
    bias = torch.cat([sd["policy_head.bias"], sd["value_head.bias"]]).double()
    z, tol = hidden @ heads.T + bias, 1040 * 2.0 ** -24 * (hidden @ heads.abs().T + bias.abs()).max()
    assert (logp.double().cpu() - torch.log_softmax(z[:, :7], 1)).abs().max() <= 2 * tol + 2.0 ** -19
    assert (value.double().cpu().reshape(-1) - torch.tanh(z[:, 7])).abs().max() <= tol + 2.0 ** -21
    p = torch.exp(logp.double().cpu()) * torch.tensor([[(int(m) >> c) & 1 for c in range(7)] for m in legal], dtype=torch.float64)
    assert (priors.double().cpu() - p / p.sum(1, keepdim=True)).abs().max() <= 2.0 ** -20


@pytest.mark.parametrize("max_games", [400, 1500])
def test_outputs_do_not_depend_on_the_batch(rp, max_games):
    """Few rows run in other forms of the kernels than many (16, 32 and 64 rows to a block, rows rounded inside the
    product's launch, tiles of 128 and 256 rows); the order of the sums goes by the engine's capacity alone."""
    import torch
    from alphazero_amd.engine import Engine
    eng = Engine(max_games=max_games, max_sims=2, precision="mx4")
    try:
        eng.load_state_dict(rp.seeded_state_dict(0))
        side, legal = _positions(eng, max_games, seed=9)
        big = eng.net_forward(side, legal)
        hidden = eng.activations(4, max_games).clone()
        for n in (1, 2, 5, 6, 16, 17, 33, 64, 65, 129, 250, max_games - 1):
            small = eng.net_forward(side[:n], legal[:n])
            for a, b in zip(big, small):
                assert torch.equal(a[:n], b), n
            assert torch.equal(eng.activations(4, n), hidden[:n]), n
    finally:
        eng.close()


@pytest.mark.parametrize("mode", ["compat", "az"])
def test_fused_and_separate_heads_agree(rp, mode):
    from alphazero_amd.engine import Engine, trajectories_to_numpy
    eng = Engine(max_games=48, max_sims=32, n_weight_sets=2, precision="mx4")
    try:
        eng.load_state_dict(rp.seeded_state_dict(0), 0)
        eng.load_state_dict(rp.seeded_state_dict(1), 1)
        n = 80                                            # more games than slots
        starters = (1 + np.arange(n) % 2).astype(np.int8)
        zeros = np.zeros((n, 2), dtype=np.uint64)
        extra = dict(dirichlet_alpha=0.3, dirichlet_eps=0.25, seed=5) if mode == "az" else {}
        for sets in ({}, {"weight_set": 0, "weight_set_colour2": 1}):
            out = []
            for separate in (False, True):
                prm = eng.params(32, 1.4, evaluator="net", mode=mode, separate_heads=separate, **extra, **sets)
                traj, stats = eng.selfplay_round(n, prm, start_boards=zeros, start_players=starters)
                out.append((trajectories_to_numpy(traj).copy(), stats))
            assert out[0][0].tobytes() == out[1][0].tobytes()
            assert out[0][1] == out[1][1]
    finally:
        eng.close()


def test_games_do_not_depend_on_slots_streams_or_cache(rp):
    from alphazero_amd.engine import Engine, trajectories_to_numpy
    out = []
    for slots in (16, 128):
        eng = Engine(max_games=slots, max_sims=32, precision="mx4", eval_cache_slots=256)
        try:
            eng.load_state_dict(rp.seeded_state_dict(0))
            kw = dict(evaluator="net", mode="az", dirichlet_alpha=0.3, dirichlet_eps=0.25, seed=3)
            for more in ({}, {"two_streams": True}, {"eval_cache": True}):
                traj, stats = eng.selfplay_round(100, eng.params(32, 1.4, **kw, **more))
                assert stats["games"] == 100
                out.append(trajectories_to_numpy(traj).tobytes())
        finally:
            eng.close()
    assert len(set(out)) == 1


def test_search_backs_up_the_value_the_network_entry_point_returns(rp):
    from alphazero_amd.engine import Engine
    from alphazero_amd.selfplay import random_openings
    eng = Engine(max_games=100, max_sims=4, precision="mx4")
    try:
        eng.load_state_dict(rp.seeded_state_dict(0), 0)
        sb, sp = random_openings(eng, 100, 6, seed=21)
        one = eng.search(sb, sp, eng.params(1, 1.4, evaluator="net", mode="compat"))
        side = np.where(sp[:, None] == 1, sb, sb[:, ::-1]).astype(np.uint64)
        _, value, _ = eng.net_forward(side)
        assert np.asarray(one[2], dtype=np.float64).tobytes() == value.cpu().numpy().astype(np.float64).tobytes()
    finally:
        eng.close()


def test_large_engine_one_and_two_streams(rp):
    """More than 1024 slots: the tiles' order of sums, two halves with buffers of their own."""
    from alphazero_amd.engine import Engine, trajectories_to_numpy
    eng = Engine(max_games=1300, max_sims=8, precision="mx4")
    try:
        eng.load_state_dict(rp.seeded_state_dict(0))
        kw = dict(evaluator="net", mode="az", lockstep=True, dirichlet_alpha=0.3, dirichlet_eps=0.25, seed=3)
        out = []
        for more in ({"one_stream": True}, {"two_streams": True}):
            traj, stats = eng.selfplay_round(1400, eng.params(8, 1.4, **kw, **more))
            assert stats["games"] == 1400
            out.append(trajectories_to_numpy(traj).tobytes())
        assert out[0] == out[1]
    finally:
        eng.close()
