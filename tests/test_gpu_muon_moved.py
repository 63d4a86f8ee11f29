"""GPU: parameters and momentum that move between two steps are written where they are, not where they were."""
import pytest
import torch

pytestmark = pytest.mark.gpu
SHAPES = [(20, 30), (3, 40, 65), (130, 70)]


def _rand(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def _grads(k):
    return [_rand(s, 10 * k + i) for i, s in enumerate(SHAPES)]


def _pair():
    """The same parameters twice: one optimizer's stay, the other's will move."""
    from mcts_q_amd.muon import DeviceMuon
    params = [[torch.nn.Parameter(_rand(s, i)) for i, s in enumerate(SHAPES)] for _ in range(2)]
    opts = [DeviceMuon(p, lr=0.1) for p in params]
    for o in opts:
        o.step(_grads(1))
    return opts


def _same(one, two):
    return all(torch.equal(a, b) for a, b in zip(one.params + one.momentum_buffers, two.params + two.momentum_buffers))


def test_parameters_move():
    stay, move = _pair()
    old = [p.data for p in move.params]
    for p in move.params:
        p.data = p.data.clone()
    kept = [t.clone() for t in old]
    for o in (stay, move):
        o.step(_grads(2))
    assert _same(stay, move) and all(torch.equal(a, b) for a, b in zip(old, kept))
    wide = torch.zeros(20, 50, device="cuda")                 # to other strides as well
    wide[:, 7:37] = move.params[0].data
    move.params[0].data = wide[:, 7:37]
    for o in (stay, move):
        o.step(_grads(3))
    assert _same(stay, move) and not wide[:, :7].any() and not wide[:, 37:].any()
    layers = torch.nn.ModuleList([torch.nn.Linear(30, 20, bias=False) for _ in range(2)]).cuda()
    from mcts_q_amd.muon import DeviceMuon
    opt = DeviceMuon([l.weight for l in layers])
    before = [l.weight.detach().clone() for l in layers]
    layers.cpu().cuda()
    opt.step([_rand((20, 30), 5), _rand((20, 30), 6)])
    assert not any(torch.equal(l.weight, b) for l, b in zip(layers, before))


def test_momentum_moves():
    stay, move = _pair()
    old = list(move.momentum_buffers)
    move.momentum_buffers[0].data = move.momentum_buffers[0].data.clone()
    move.momentum_buffers[1] = move.momentum_buffers[1].clone()
    kept = old[1].clone()
    for o in (stay, move):
        o.step(_grads(2))
    assert _same(stay, move) and torch.equal(old[1], kept)


def test_moves_that_no_step_can_follow():
    from mcts_q_amd import MctsqError
    for spoil in (lambda o: setattr(o.params[0], "data", o.params[0].data.bfloat16()),
                  lambda o: setattr(o.params[0], "data", o.params[0].data.t().contiguous().t()),
                  lambda o: setattr(o.params[0], "data", o.params[0].data[:10].clone()),
                  lambda o: setattr(o.params[0], "data", o.momentum_buffers[0]),
                  lambda o: setattr(o.params[0], "data", o.params[2].data.view(-1)[:600].view(20, 30)),
                  lambda o: setattr(o.params[0], "data", o.params[0].data.cpu()),
                  lambda o: o.momentum_buffers.__setitem__(0, o.momentum_buffers[0][:, :20])):
        _, opt = _pair()
        spoil(opt)
        kept = [t.clone() for t in opt.params + opt.momentum_buffers]
        for _ in range(2):
            with pytest.raises((ValueError, MctsqError)):
                opt.step([_rand(p.shape, 4) for p in opt.params])
        assert all(torch.equal(a, b) for a, b in zip(kept, opt.params + opt.momentum_buffers))


def test_a_gradient_that_a_parameter_moved_onto():
    _, opt = _pair()
    grads = _grads(2)
    opt.params[0].data = grads[0]
    with pytest.raises(ValueError, match=r"grads\[0\]"):
        opt.step(grads)
