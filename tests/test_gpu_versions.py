"""GPU: autograd, and a network that prepared something from its weights, are told of what the kernels write."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def test_a_step_between_forward_and_backward_is_caught():
    from mcts_q_amd.muon import DeviceMuon
    p = torch.nn.Parameter(_rand((20, 30), 1))
    loss = (p * p).sum()                                    # the product's backward reads p
    DeviceMuon([p]).step([_rand((20, 30), 2)])
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    m = torch.zeros(20, 30, device="cuda", requires_grad=True)
    q = m * 1.0                                             # momentum that somebody's graph still needs
    r = (q * q).sum()
    DeviceMuon([p], momentum_buffers=[q.detach()]).step([_rand((20, 30), 3)])
    with pytest.raises(RuntimeError, match="inplace"):
        r.backward()


def test_a_gradient_over_saved_logits_is_caught():
    from mcts_q_amd.muon import orthogonalize
    from mcts_q_amd.policyloss import policy_loss, preference_loss
    x = _rand((4, 6, 10), 3).requires_grad_(True)
    a = torch.zeros(4, 6, dtype=torch.int64, device="cuda")
    for write in (lambda z: policy_loss(z, a, None, torch.ones(4, 6, device="cuda"), out=z),
                  lambda z: preference_loss(z, a, torch.zeros(4, device="cuda"), out=z),
                  lambda z: orthogonalize(z, out=z)):
        z = x.exp()                                         # its backward reads its result
        write(z.detach())
        with pytest.raises(RuntimeError, match="inplace"):
            z.sum().backward()
    z = x.exp()                                             # nothing is written: nothing to catch
    policy_loss(z.detach(), a, None, torch.ones(4, 6, device="cuda"))
    orthogonalize(z.detach())
    z.sum().backward()


def test_a_network_sees_its_weights_move():
    """Parameters that are views of a network's flat buffer: the next evaluation multiplies by the new weights."""
    from mcts_q_amd import NetSpec
    from mcts_q_amd.muon import DeviceMuon
    from mcts_q_amd.qnet import DeviceQNet
    net = DeviceQNet(NetSpec.from_cfg(dict(price="gru", process="gru", gas="gru", act="relu", flavor="per")))
    net.flat.copy_(_rand((net.n_flat,), 4) * 0.1)
    state = torch.rand(7, 25, 1, device="cuda"), torch.rand(7, 10, 6, device="cuda"), torch.rand(7, 3, 2, device="cuda")
    before = net(*state)["q"].clone()
    views = net.views()
    keys = [k for k, v in views.items() if v.dim() == 2 and min(v.shape) >= 16]
    DeviceMuon([views[k] for k in keys], lr=0.3).step([_rand(views[k].shape, 5 + i) for i, k in enumerate(keys)])
    after = net(*state)["q"].clone()
    net.mark_dirty()
    assert torch.equal(after, net(*state)["q"]) and not torch.equal(after, before)


def test_inference_tensors_are_taken():
    """They carry no version: nothing to tell, the calls work."""
    from mcts_q_amd.muon import DeviceMuon, orthogonalize
    from mcts_q_amd.policyloss import policy_loss
    with torch.inference_mode():
        p, z = _rand((20, 30), 1), _rand((4, 10), 2)
        a = torch.zeros(4, dtype=torch.int64, device="cuda")
        want = policy_loss(z, a, None, torch.ones(4, device="cuda"))["dlogits"]
        policy_loss(z, a, None, torch.ones(4, device="cuda"), out=z)
        assert torch.equal(z, want)
        orthogonalize(p, out=p)
        before = p.clone()
        DeviceMuon([p]).step([_rand((20, 30), 3)])
        assert not torch.equal(p, before)
