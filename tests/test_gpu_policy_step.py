"""GPU: the policy losses and the Muon step as they are used together, and Muon inside the agent's learner."""
import math

import numpy as np
import pytest
import torch

from oracle import torch_ref

pytestmark = pytest.mark.gpu
COEF = (3.4445, -4.7750, 2.0315)
TOL = 200 * 8 * 2.0 ** -23             # of an orthogonalised fp32 matrix (tests/test_gpu_muon.py: its derivation)


def _orth64(x):
    x = x.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / (x.norm() + 1e-7)
    for _ in range(5):
        s = x @ x.t()
        x = COEF[0] * x + (COEF[1] * s + COEF[2] * (s @ s)) @ x
    return x.t().contiguous() if tall else x


def test_policy_and_preference_steps_of_a_head():
    """A linear head: behaviour and reference log-probabilities, a clipped policy step, then a preference step, each
    gradient through the head's product into a Muon step; against the same in 64 bits with autograd.

    The products around the operators are torch's in fp32: a gradient element is a sum of N = 480 of them, off by at most
    N 2^-24 of its terms' size, and the orthogonalisation lets that grow 200 times at most."""
    from mcts_q_amd.muon import DeviceMuon
    from mcts_q_amd.policyloss import policy_loss, preference_loss, token_logprobs
    g = torch.Generator(device="cuda").manual_seed(31)
    P, T, V, D = 8, 30, 64, 96
    x = torch.randn(2 * P, T, D, generator=g, device="cuda")
    W0 = torch.randn(V, D, generator=g, device="cuda") * 0.1
    Wref = W0 + 0.02 * torch.randn(V, D, generator=g, device="cuda")
    a = torch.randint(0, V, (2 * P, T), generator=g, device="cuda")
    mask = (torch.rand(2 * P, T, generator=g, device="cuda") < 0.8).float()
    mask[:, 0] = 1
    a = torch.where(mask != 0, a, -1)
    adv = torch.randn(2 * P, generator=g, device="cuda")
    w = mask / mask.sum()
    flat = x.view(-1, D)
    W = W0.clone()
    opt = DeviceMuon([W], lr=0.05, momentum=0.9)
    old, ref = token_logprobs(x @ W.t(), a, weight=mask), token_logprobs(x @ Wref.t(), a, weight=mask)
    r = policy_loss(x @ W.t(), a, old, adv, ref_logp=ref, weight=w, kl_coef=0.1)
    opt.step([r["dlogits"].view(-1, V).t() @ flat])
    W1 = W.clone()
    z = x @ W.t()
    q = preference_loss(z, a, (mask * ref).sum(1), weight=mask, beta=0.2, out=z)        # the gradient over the logits
    opt.step([z.view(-1, V).t() @ flat])

    x64, live = x.double(), mask != 0

    def logp(W):
        return torch.where(live, torch.log_softmax(x64 @ W.t(), -1).gather(-1, a.clamp(min=0)[..., None])[..., 0], 0.0)

    def moved(W, m, grad, lr=0.05):
        m = 0.9 * m + grad
        return W - lr * math.sqrt(max(1.0, V / D)) * _orth64(grad + 0.9 * m), m

    Wd = W0.double().requires_grad_(True)
    lp, rf = logp(Wd), logp(Wref.double()).detach()
    ratio = (lp - lp.detach()).exp()
    A = adv.double()[:, None]
    loss = (w.double() * (-torch.minimum(ratio * A, ratio.clamp(0.8, 1.2) * A) + 0.1 * ((rf - lp).exp() - (rf - lp) - 1)))[live].sum()
    loss.backward()
    tol = TOL + 200 * 480 * 2.0 ** -24
    assert abs(float(r["loss"]) - float(loss.detach())) <= 480 * 2.0 ** -24 * float((w * adv.abs()[:, None]).sum() + 1)
    W1d, m = moved(Wd.detach(), torch.zeros_like(Wd), Wd.grad)
    step = (W1d - W0.double()).norm()
    assert (W1.double() - W1d).norm() <= tol * step
    W1d = W1.double().requires_grad_(True)                       # the second step from where the first one really ended
    S = (mask.double() * logp(W1d)).sum(1)
    R = (mask.double() * rf).sum(1)
    h = 0.2 * ((S[:P] - R[:P]) - (S[P:] - R[P:]))
    loss = -torch.nn.functional.logsigmoid(h).mean()
    loss.backward()
    assert abs(float(q["loss"]) - float(loss.detach())) <= 0.2 * 2 * T * 480 * 2.0 ** -24 + 2.0 ** -23
    W2d, _ = moved(W1d.detach(), m, W1d.grad)
    assert (W.double() - W2d).norm() <= tol * (W2d - W1d).norm() + tol * step


def _learners(combo=("gru", "gru", "gru")):
    from mcts_q_amd import NetSpec
    from mcts_q_amd.learner import DeviceLearner
    cfg = dict(price=combo[0], process=combo[1], gas=combo[2], act="relu", flavor="per")
    torch.manual_seed(5)
    sd = {k: v.detach().numpy() for k, v in torch_ref.RefQNet(cfg).state_dict().items()}
    spec = NetSpec.from_cfg(cfg)
    return DeviceLearner(spec).load_state_dict(sd), DeviceLearner(spec, optimizer="muon", muon_lr=0.01).load_state_dict(sd)


def _replay():
    from mcts_q_amd.per import DevicePER
    rng = np.random.RandomState(3)
    buf = DevicePER(2048)
    n = 1500
    rows, nxt = rng.standard_normal((2, n, 91)).astype(np.float32)
    buf.push_rows(rows, rng.randint(0, 5, n), rng.standard_normal(n), nxt, (rng.random_sample(n) < 0.1).astype(np.float64))
    return buf


@pytest.mark.parametrize("combo", [("gru", "gru", "gru"), ("conv", "gru", "mlp"), ("transformer", "gru", "mlp")])
def test_learner_moves_matrices_by_muon_and_the_rest_by_adam(combo):
    adam, muon = _learners(combo)
    buf = _replay()
    u = np.random.RandomState(4).random_sample(256)
    batch, w, _, _ = buf.sample_batch(u)
    for L in (adam, muon):
        L.compute_grad(batch, w)
    assert torch.equal(adam.grad, muon.grad)
    before = {k: v.clone() for k, v in muon.policy.views().items()}
    target = muon.target.flat.clone()
    for L in (adam, muon):
        L.apply_grad(tau=0.25)
    va, vm, gr = adam.policy.views(), muon.policy.views(), muon.policy.views(muon.grad)
    keys = muon.muon_keys()
    assert keys and torch.equal(adam.grad_norm, muon.grad_norm)
    for k in vm:
        if k in keys:
            m = gr[k].double()                                   # momentum starts at 0
            r, c = m.shape
            want = before[k].double() - 0.01 * math.sqrt(max(1.0, r / c)) * _orth64(m + 0.95 * m)
            err = (vm[k].double() - want).norm()
            assert err <= TOL * (want - before[k].double()).norm() + 2.0 ** -23 * want.norm(), k
        else:
            assert torch.equal(vm[k], va[k]), k                  # the same kernel, the same norm
    assert torch.allclose(muon.target.flat, 0.25 * muon.policy.flat + 0.75 * target, rtol=1e-6, atol=1e-9)
    # a leaf evaluation right behind the step sees the new weights
    p, c, gs = torch.rand(7, 25, 1).cuda(), torch.rand(7, 10, 6).cuda(), torch.rand(7, 3, 2).cuda()
    q = muon.policy(p, c, gs)["q"].clone()
    muon.policy.mark_dirty()
    assert torch.equal(q, muon.policy(p, c, gs)["q"])


def test_agent_update_with_muon_and_its_checkpoint(tmp_path):
    """DQNModel(optimizer="muon"): update() as with Adam; a saved and reloaded model makes the same next step."""
    from mcts_q_amd import MctsqError
    from mcts_q_amd.dqn import DQNModel
    args = dict(el_input_dim=1, process_input_dim=6, gas_eua_input_dim=2, action_dim=5, embed_dim=64, hidden_layers=2,
                hidden_units=128, buffer_capacity=512, batch_size=64, gamma=0.99, lr=1e-3, price_encoder_type="gru",
                process_encoder_type="gru", gas_eua_encoder_type="gru", learning_starts=64)
    a = DQNModel(**args, seed=7, optimizer="muon")
    rng = np.random.RandomState(6)
    rows, nxt = rng.standard_normal((2, 300, 91)).astype(np.float32)
    a.replay_buffer.dev.push_rows(rows, rng.randint(0, 5, 300), rng.standard_normal(300), nxt, np.zeros(300))
    start = a.learner.policy.flat.clone()
    for _ in range(3):
        a.learner.step(a.replay_buffer.dev, rng.random_sample(64), tau=0.005)
        assert torch.isfinite(a.learner.loss).all() and float(a.learner.loss) > 0
    assert not torch.equal(start, a.learner.policy.flat)
    state = a.optimizer.state_dict()
    b = DQNModel(**args, seed=8, optimizer="muon")
    b.learner.policy.flat.copy_(a.learner.policy.flat)
    b.learner.target.flat.copy_(a.learner.target.flat)
    b.optimizer.load_state_dict(state)
    batch, w, _, _ = a.replay_buffer.dev.sample_batch(rng.random_sample(64))
    for m in (a, b):
        m.learner.compute_grad(batch, w)
        m.learner.apply_grad(tau=0.005)
    assert torch.equal(a.learner.policy.flat, b.learner.policy.flat) and torch.equal(a.learner.target.flat, b.learner.target.flat)
    with pytest.raises(ValueError):
        DQNModel(**args, optimizer="sgd")
    with pytest.raises(MctsqError):
        a.learner.step_sharded(a.replay_buffer.dev, rng.random_sample(8))
