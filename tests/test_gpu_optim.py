"""Orthogonalisation and the optimiser step against their formulas in float64."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# Operands carry 22 bits and sums are float32: a product is off by at most 2^-20 of its factors' norms.  Such an error in
# A = X X^T grows by a^2 a step in the directions of small singular values, twice before X is looked at again, enters
# p(A) with the factor |b| against a: 2^-20 |b| a^4 / a relative to those directions, once per segment of steps.
FAITHFUL = 2 * 2.0 ** -20 * abs(B) * A ** 3


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X (torch.cuda.is_available() is False)")
    return torch


def orthogonalized(x, steps=5, coefficients=(A, B, C), eps=1e-7):
    """x numpy float64 [rows, cols], by the formula."""
    x = x / (np.sqrt((x * x).sum()) + eps)
    rows = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else coefficients
    for a, b, c in rows:
        tall = x.shape[0] > x.shape[1]
        g = x.T @ x if tall else x @ x.T
        q = b * g + c * (g @ g)
        x = a * x + (x @ q if tall else q @ x)
    return x


def _check(got, want, dtype, extra=0.0):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    size = np.sqrt((want * want).sum())
    # one rounding to the type (a half's smallest step is 2^-24), in the Frobenius norm
    tol = (FAITHFUL + HALF_STEP[dtype] + extra) * size + (2.0 ** -25 * math.sqrt(want.size) if dtype == "float16" else 0.0)
    err = np.sqrt(((got - want) ** 2).sum())
    assert err <= tol, (err / max(size, 1e-300), tol / max(size, 1e-300))


def _gradient(shape, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    return x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g)) * 1e-3


SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (5, 300), (300, 5), (31, 33), (64, 64), (63, 65), (65, 64), (128, 32), (7, 1024),
          (100, 1000), (129, 515), (515, 129), (200, 200), (256, 257), (128, 2048), (700, 333)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize_against_float64(shape, dtype):
    torch = _torch()
    from alphazero_amd import optim
    x = _gradient(shape, shape[0] * 1009 + shape[1]).to(getattr(torch, dtype))
    got = optim.orthogonalize(x.cuda())
    assert got.dtype == x.dtype
    _check(got, orthogonalized(x.double().numpy()), dtype)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 10])
def test_other_step_counts(steps):
    torch = _torch()
    from alphazero_amd import optim
    for shape in ((96, 160), (20, 24)):
        x = _gradient(shape, steps)
        _check(optim.orthogonalize(x.cuda(), steps=steps), orthogonalized(x.double().numpy(), steps), "float32")


def test_other_coefficients():
    torch = _torch()
    from alphazero_amd import optim
    x = _gradient((150, 260), 3)
    for coefficients, steps in (((1.5, -0.5, 0.0), 8), ((15 / 8, -10 / 8, 3 / 8), 8), ((2.0, -1.5, 0.5), 5), ((1.0, 0.0, 0.0), 3),
                                ([(4.0, -6.0, 2.5), (3.0, -3.0, 1.0), (1.875, -1.25, 0.375)], 3)):
        got = optim.orthogonalize(x.cuda(), steps=steps, coefficients=coefficients)
        _check(got, orthogonalized(x.double().numpy(), steps, coefficients), "float32")


def test_ill_conditioned_matrices():
    """Rank 8 of 128, and singular values over six decades."""
    torch = _torch()
    from alphazero_amd import optim
    r = np.random.default_rng(1)
    low = r.standard_normal((128, 8)) @ r.standard_normal((8, 500))
    u, v = np.linalg.qr(r.standard_normal((160, 160)))[0], np.linalg.qr(r.standard_normal((400, 160)))[0]
    decades = u @ np.diag(10.0 ** np.linspace(0, -6, 160)) @ v.T
    for x in (low, decades, decades.T.copy()):
        x = torch.from_numpy(x).float()
        _check(optim.orthogonalize(x.cuda()), orthogonalized(x.double().numpy()), "float32")


def test_result_is_nearly_orthogonal():
    """The quintic leaves singular values between about 0.7 and 1.2 (one of its fixed intervals is [0.68, 1.13])."""
    torch = _torch()
    from alphazero_amd import optim
    got = optim.orthogonalize(torch.randn(200, 900, generator=torch.Generator().manual_seed(2)).cuda())
    s = np.linalg.svd(got.double().cpu().numpy(), compute_uv=False)
    assert s.min() > 0.6 and s.max() < 1.3


@pytest.mark.parametrize("magnitude", [1e-30, 1e-12, 1e12, 1e30])
def test_magnitudes_whose_squares_leave_float32(magnitude):
    torch = _torch()
    from alphazero_amd import optim
    for shape in ((40, 90), (90, 200)):
        x = (torch.randn(shape, generator=torch.Generator().manual_seed(4)).double() * magnitude).float()
        _check(optim.orthogonalize(x.cuda(), eps=0.0), orthogonalized(x.double().numpy(), eps=0.0), "float32")


def test_zero_nan_and_infinity():
    torch = _torch()
    from alphazero_amd import optim
    for shape in ((30, 50), (70, 150), (150, 70)):
        x = torch.randn(4, *shape, generator=torch.Generator().manual_seed(5))
        x[0] = 0.0
        x[1, 3, 4], x[2, 7, 1] = float("nan"), float("inf")
        got = optim.orthogonalize(x.cuda())
        assert not got[0].any() and got[1].isnan().all() and got[2].isnan().all()
        _check(got[3], orthogonalized(x[3].double().numpy()), "float32")        # its neighbours do not touch it


def test_batches_strides_and_out():
    torch = _torch()
    from alphazero_amd import optim
    base = _gradient((6, 90, 140), 6).cuda()
    views = [base, base.transpose(1, 2), base[:, 3:80, 5:120], base[::2, ::2, ::3], base.reshape(2, 3, 90, 140), base[4],
             base[:1].expand(3, 90, 140), base.flip(2), base.bfloat16()[:, :, 1:], base[:0], base[:, :0], base[:, :, :0]]
    for v in views:
        got = optim.orthogonalize(v)
        assert got.shape == v.shape and got.dtype == v.dtype
        if v.numel():
            x = v.double().cpu().numpy().reshape((-1,) + tuple(v.shape[-2:]))
            for i, y in enumerate(got.reshape((-1,) + tuple(v.shape[-2:]))):
                _check(y, orthogonalized(x[i]), str(v.dtype).split(".")[1])
    want = optim.orthogonalize(base)
    wide = torch.full((6, 100, 150), 7.0, device="cuda")
    got = optim.orthogonalize(base, out=wide[:, 5:95, 4:144])
    assert torch.equal(got, want)
    wide[:, 5:95, 4:144] = 7.0
    assert (wide == 7.0).all()                                                  # nothing beside the result was written
    x = base.clone()
    assert optim.orthogonalize(x, out=x) is x and torch.equal(x, want)
    assert torch.equal(optim.orthogonalize(base), want)                         # the same call gives the same bits
    assert torch.equal(optim.orthogonalize(base[2]), want[2])                   # whatever stands beside a matrix


def _muon_reference(w, g, m, lr, mu, nesterov, wd, steps=5):
    w, g, m = (t.double().cpu().reshape(t.shape[0], -1).numpy() for t in (w, g, m))
    m = mu * m + g
    u = g + mu * m if nesterov else m
    o = orthogonalized(u, steps)
    scale = lr * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
    return w * (1.0 - lr * wd) - scale * o, m, scale * o


NETWORK = [(128, 2, 4, 4), (128, 128, 4, 4), (128, 128, 4, 4), (512, 3000)]
MANY = [(1 + 7 * i % 90, 1 + 13 * i % 150) for i in range(50)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shapes", [NETWORK, MANY, [(33, 70)]], ids=["network", "many", "one"])
def test_muon_update_against_float64(shapes, dtype, nesterov):
    torch = _torch()
    from alphazero_amd import optim
    g = torch.Generator().manual_seed(len(shapes))
    dt = getattr(torch, dtype)
    grads = [_gradient(s, i).to(dt).cuda() for i, s in enumerate(shapes)]
    weights = [(torch.randn(s, generator=g) / 10).to(dt).cuda() for s in shapes]
    momenta = [(torch.randn(s, generator=g) * 1e-3).cuda() for s in shapes]
    kept = [t.clone() for t in weights + momenta]
    kw = dict(lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    new_w, new_m = optim.muon_update(weights, grads, momenta, inplace=False, **kw)
    assert all(torch.equal(a, b) for a, b in zip(weights + momenta, kept))
    for w, gr, m, w2, m2 in zip(weights, grads, momenta, new_w, new_m):
        want_w, want_m, move = _muon_reference(w, gr, m, 0.05, 0.9, nesterov, 0.1)
        got_m = m2.double().cpu().numpy().reshape(want_m.shape)
        # two roundings, of 0.9 as a float32, of the product and of the sum
        tol = 4 * 2.0 ** -24 * (np.abs(0.9 * m.double().cpu().numpy()) + np.abs(gr.double().cpu().numpy())).reshape(want_m.shape)
        assert (np.abs(got_m - want_m) <= tol + 1e-45).all()
        got_w = w2.double().cpu().numpy().reshape(want_w.shape)
        err = np.sqrt(((got_w - want_w) ** 2).sum())
        size = np.sqrt((want_w ** 2).sum())
        tol = FAITHFUL * np.sqrt((move ** 2).sum()) + (HALF_STEP[dtype] + 8 * 2.0 ** -24) * size
        if dtype == "float16":
            tol += 2.0 ** -25 * math.sqrt(want_w.size)
        assert err <= tol, (w.shape, err / size)
    got_w, got_m = optim.muon_update(weights, grads, momenta, **kw)             # in place: the same bits
    assert got_w[0] is weights[0] and got_m[0] is momenta[0]
    assert all(torch.equal(a, b) for a, b in zip(weights + momenta, list(new_w) + list(new_m)))


def test_muon_empty_matrices_and_empty_lists():
    torch = _torch()
    from alphazero_amd import optim
    assert optim.muon_update([], [], [], lr=0.1) == ([], [])
    z = lambda *s: torch.zeros(s, device="cuda")
    optim.muon_update([z(0, 5), z(4, 0)], [z(0, 5), z(4, 0)], [z(0, 5), z(4, 0)], lr=0.1)
    w = torch.randn(8, 9, generator=torch.Generator().manual_seed(1)).cuda()
    before = w.clone()
    optim.muon_update([z(0, 5), w], [z(0, 5), z(8, 9)], [z(0, 5), z(8, 9)], lr=0.1)
    assert torch.equal(w, before)                                               # a zero gradient moves nothing


def test_muon_optimizer_trains_the_network_and_the_engine_sees_it():
    """Samples -> gradients -> Muon + Adam -> the engine evaluates the new weights: the parts used together."""
    torch = _torch()
    from alphazero_amd import optim
    from alphazero_amd.agent import initialize_agent
    from alphazero_amd.selfplay import self_play_sample_tensors
    torch.manual_seed(0)
    agent = initialize_agent(use_gpu=True, num_simulations=16, load_model=False)
    planes, probs, z = self_play_sample_tensors(agent, 4)
    matrices, rest = optim.split_parameters(agent.model)
    assert [tuple(p.shape) for p in matrices] == [(128, 2, 4, 4), (128, 128, 4, 4), (128, 128, 4, 4), (1024, 11520)]
    assert len(rest) == 8
    muon, adam = optim.Muon(matrices, lr=0.02, weight_decay=0.01), torch.optim.Adam(rest, lr=1e-3)
    want = [(p.detach().clone(), torch.zeros_like(p)) for p in matrices]
    for step in range(2):
        logp, value = agent.model(planes)
        loss = torch.nn.functional.kl_div(logp, probs, reduction="batchmean") + torch.nn.functional.mse_loss(value[:, 0], z)
        muon.zero_grad()
        adam.zero_grad()
        loss.backward()
        grads = [p.grad.clone() for p in matrices]
        versions = [p._version for p in matrices]
        muon.step()
        adam.step()
        assert all(p._version > v for p, v in zip(matrices, versions))
        for i, p in enumerate(matrices[:3]):                                    # the large one is checked elsewhere
            w, m, move = _muon_reference(want[i][0], grads[i], want[i][1], 0.02, 0.95, True, 0.01)
            got = p.detach().double().cpu().numpy().reshape(w.shape)
            assert np.sqrt(((got - w) ** 2).sum()) <= FAITHFUL * np.sqrt((move ** 2).sum()) + 2.0 ** -21 * np.sqrt((w ** 2).sum())
            want[i] = (p.detach().clone(), muon.state[p]["momentum"].clone())
    eng = agent.engine(1)
    logp_e, value_e = eng.net_forward_planes(planes[:4])
    with torch.no_grad():
        logp, value = agent.model.cpu()(planes[:4].cpu())
    assert (logp_e.cpu() - logp).abs().max() < 1e-4 * (1 + logp.abs().max()) and (value_e.cpu() - value).abs().max() < 1e-4


def test_muon_state_dict_keeps_float32_momentum():
    torch = _torch()
    from alphazero_amd import optim
    p = torch.nn.Parameter(torch.randn(20, 30, generator=torch.Generator().manual_seed(3)).bfloat16().cuda())
    p.grad = torch.ones_like(p)
    opt = optim.Muon([p], lr=0.1)
    opt.step()
    q = torch.nn.Parameter(p.detach().clone())
    q.grad = p.grad.clone()
    other = optim.Muon([q], lr=0.1)
    other.load_state_dict(opt.state_dict())
    assert other.state[q]["momentum"].dtype == torch.float32
    assert torch.equal(other.state[q]["momentum"], opt.state[p]["momentum"])
    opt.step()
    other.step()
    assert torch.equal(p, q)
    assert other.state[q]["momentum"].data_ptr() != opt.state[p]["momentum"].data_ptr()


def test_streams_and_graph():
    torch = _torch()
    from alphazero_amd import optim
    shapes = [(128, 32), (128, 300), (90, 500)]
    grads = [_gradient(s, i).cuda() for i, s in enumerate(shapes)]
    start = [torch.randn(s, generator=torch.Generator().manual_seed(i)).cuda() for i, s in enumerate(shapes)]
    zero = [torch.zeros_like(w) for w in start]
    eager_w, eager_m = [w.clone() for w in start], [m.clone() for m in zero]
    history = []
    for k in range(4):
        optim.muon_update(eager_w, [g * (k + 1) for g in grads], eager_m, lr=0.1)
        history.append([w.clone() for w in eager_w])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w, m = [t.clone() for t in start], [t.clone() for t in zero]
        optim.muon_update(w, grads, m, lr=0.1)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(w, history[0]))
    w, m, gs = [t.clone() for t in start], [t.clone() for t in zero], [g.clone() for g in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.muon_update(w, gs, m, lr=0.1)
    for k in range(4):
        for a, b in zip(gs, grads):
            a.copy_(b * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(w, history[k]))
        optim.orthogonalize(grads[0])                                           # eager work between the replays
    torch.cuda.synchronize()


def test_two_streams_at_once():
    torch = _torch()
    from alphazero_amd import optim
    x = [_gradient((200, 400), i).cuda() for i in range(2)]
    want = [optim.orthogonalize(t) for t in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(optim.orthogonalize(x[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
