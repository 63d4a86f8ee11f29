"""GPU: what DQNModel.save writes of a Muon optimizer, and which optimizer takes it back."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ARGS = dict(el_input_dim=1, process_input_dim=6, gas_eua_input_dim=2, action_dim=5, embed_dim=64, hidden_layers=2,
            hidden_units=128, buffer_capacity=512, batch_size=64, gamma=0.99, lr=1e-3, price_encoder_type="gru",
            process_encoder_type="gru", gas_eua_encoder_type="gru", learning_starts=64)


def _model(optimizer, seed=7, steps=3):
    from mcts_q_amd.dqn import DQNModel
    m = DQNModel(**ARGS, seed=seed, optimizer=optimizer)
    rng = np.random.RandomState(6)
    rows, nxt = rng.standard_normal((2, 300, 91)).astype(np.float32)
    m.replay_buffer.dev.push_rows(rows, rng.randint(0, 5, 300), rng.standard_normal(300), nxt, np.zeros(300))
    for _ in range(steps):
        loss = m.update()
        assert torch.isfinite(loss) and float(loss) > 0
        m.update_target_network(0.005)
    return m


def _everything(m):
    L = m.learner
    return [t.clone() for t in (L.policy.flat, L.target.flat, L.exp_avg, L.exp_avg_sq)] + [
        L.step_count, L.lr, L.betas, L.eps, len(m.replay_buffer)] + (
        [L.muon.lr, L.muon.momentum] if L.optimizer == "muon" else [])


def _same(a, b):
    return all(torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(a, b, strict=True))


@pytest.mark.parametrize("optimizer", ["adam", "muon"])
def test_saved_and_loaded_training_goes_on(optimizer, tmp_path):
    """Through save() and load() into a model of other weights: the next update() is the same, bit for bit."""
    a, b = _model(optimizer), _model(optimizer, seed=8, steps=1)
    if optimizer == "muon":
        a.learner.muon.lr, a.learner.muon.momentum = 0.015, 0.9
    f = str(tmp_path / "c.pt")
    a.save(f)
    b.load(f)
    assert _same(_everything(a), _everything(b))
    for m in (a, b):
        np.random.seed(3)
        m.update()
        m.update_target_network(0.005)
    assert _same(_everything(a), _everything(b))


@pytest.mark.parametrize("writer,reader", [("muon", "adam"), ("adam", "muon")])
def test_the_other_optimizer_refuses_it_and_stays_as_it_was(writer, reader, tmp_path):
    a, b = _model(writer), _model(reader, seed=8)
    f = str(tmp_path / "c.pt")
    a.save(f)
    before = _everything(b)
    with pytest.raises(ValueError, match="Muon"):
        b.load(f)
    assert _same(before, _everything(b))
    with pytest.raises(ValueError, match="Muon"):
        b.optimizer.load_state_dict(a.optimizer.state_dict())
    assert _same(before, _everything(b))


def test_momentum_in_adams_layout_is_told_by_its_values():
    """A file of the layout that wrote Muon's momentum as exp_avg, exp_avg_sq 0, under one parameter group: Adam refuses it
    (its own first moment cannot be nonzero where the second is 0), Muon takes it."""
    a, adam, muon = _model("muon"), _model("adam", seed=8), _model("muon", seed=9)
    L = a.learner
    m, v = L.policy.views(L.exp_avg), L.policy.views(L.exp_avg_sq)
    old = {"state": {i: {"step": torch.tensor(float(L.step_count)), "exp_avg": m[k].cpu().clone(),
                         "exp_avg_sq": v[k].cpu().clone()} for i, k in enumerate(m)},
           "param_groups": [{"lr": L.lr, "betas": tuple(L.betas), "eps": L.eps, "params": list(range(len(m)))}]}
    before = _everything(adam)
    with pytest.raises(ValueError, match="Muon"):
        adam.optimizer.load_state_dict(old)
    assert _same(before, _everything(adam))
    muon.optimizer.load_state_dict(old)
    assert torch.equal(muon.learner.exp_avg, L.exp_avg) and torch.equal(muon.learner.exp_avg_sq, L.exp_avg_sq)
    assert muon.learner.step_count == 3


def test_torchs_adam_does_not_take_it():
    """A reader outside: torch.optim.Adam over the same parameters refuses the state instead of dividing by nothing."""
    a = _model("muon")
    params = [torch.nn.Parameter(v.clone()) for v in a.learner.policy.views().values()]
    with pytest.raises((ValueError, KeyError)):
        opt = torch.optim.Adam(params)
        opt.load_state_dict(a.optimizer.state_dict())
        for p in params:
            p.grad = torch.ones_like(p)
        opt.step()
    b = _model("adam")
    opt = torch.optim.Adam(params)
    opt.load_state_dict(b.optimizer.state_dict())
    for p in params:
        p.grad = torch.zeros_like(p)
    opt.step()


def test_before_the_first_step():
    """No state yet: a fresh model's file loads into its own kind, and an Adam file without state into either."""
    fresh = _model("adam", steps=0)
    for optimizer in ("adam", "muon"):
        m = _model(optimizer, seed=8, steps=1)
        m.optimizer.load_state_dict(fresh.optimizer.state_dict())
        assert m.learner.step_count == 0 and not m.learner.exp_avg.any()
    one, two = _model("muon", steps=0), _model("muon", seed=8, steps=1)
    two.optimizer.load_state_dict(one.optimizer.state_dict())
    assert two.learner.step_count == 0 and not two.learner.exp_avg.any()


def test_adam_state_in_several_groups():
    """Only the mark makes a group Muon's: an Adam state of two groups is Adam's, its first group gives the settings."""
    a, b = _model("adam"), _model("adam", seed=8)
    sd = a.optimizer.state_dict()
    n = len(sd["param_groups"][0]["params"])
    sd["param_groups"] = [dict(sd["param_groups"][0], params=list(range(n // 2))),
                          dict(sd["param_groups"][0], params=list(range(n // 2, n)), lr=0.5)]
    b.optimizer.load_state_dict(sd)
    assert torch.equal(a.learner.exp_avg, b.learner.exp_avg) and torch.equal(a.learner.exp_avg_sq, b.learner.exp_avg_sq)
    assert b.learner.step_count == 3 and b.learner.lr == 1e-3
    with pytest.raises(ValueError, match="Muon"):
        _model("muon", seed=9, steps=1).optimizer.load_state_dict(sd)
