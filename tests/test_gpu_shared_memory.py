"""GPU: strided tensors that share memory with what a call writes are refused; interleaved ones that share none are not."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def test_parameters_that_cross():
    from mcts_q_amd.muon import DeviceMuon
    wide = torch.zeros(6, 20, device="cuda")
    ones = [torch.zeros(6, 8, device="cuda") for _ in range(2)]
    for params in ([wide[:, :8], wide[:, 4:12]], [wide[:, :8], wide[2:4]], [wide[2:4], wide[:, :8]], [wide[:, 2:10], wide[:4, :8]],
                   [wide[:3, :8], wide[2:, :8]]):
        with pytest.raises(ValueError, match="share memory"):
            DeviceMuon(params)
    # momentum inside a strided parameter's rows
    flat = torch.zeros(400, device="cuda")
    param = flat[:320].view(8, 40)[:, :20]
    for m in (flat[10:170].view(8, 20), flat[100:260].view(8, 20)):
        with pytest.raises(ValueError, match="momentum"):
            DeviceMuon([param], momentum_buffers=[m])
    opt = DeviceMuon([wide[:, :8], wide[:, 8:16]], momentum_buffers=ones)
    for bad in (wide[:, 4:12], wide[:, 1:9], wide[:, 12:20], wide.view(-1)[4:52].view(6, 8)):
        with pytest.raises(ValueError, match=r"grads\[1\]"):
            opt.step([_rand((6, 8), 1), bad])
    assert not wide.any() and not ones[0].any() and not ones[1].any()


def test_parameters_and_gradients_in_turn():
    """Columns of one buffer, and stacks whose matrices lie row by row between each other: the results of separate ones."""
    from mcts_q_amd.muon import DeviceMuon, orthogonalize
    wide = torch.full((70, 200), 3.0, device="cuda")
    a, b, ga, gb = wide[:, :60], wide[:, 61:100], wide[:, 100:160], wide[:, 160:199]
    stack = torch.zeros(40, 3, 33, device="cuda").transpose(0, 1)       # [3, 40, 33], row r of every matrix side by side
    gs = torch.zeros(40, 3, 33, device="cuda").transpose(0, 1)
    want = [_rand(t.shape, 1 + i) for i, t in enumerate((a, b, stack))]
    grads = [_rand(t.shape, 11 + i) for i, t in enumerate((a, b, stack))]
    for t, w in zip((a, b, stack, ga, gb, gs), want + grads):
        t.copy_(w)
    one, two = DeviceMuon([a, b, stack], weight_decay=0.1), DeviceMuon(want, weight_decay=0.1)
    for _ in range(2):
        one.step([ga, gb, gs])
        two.step(grads)
    assert all(torch.equal(t, w) for t, w in zip((a, b, stack, ga, gb, gs), want + grads))
    assert (wide[:, 60] == 3).all() and (wide[:, 199] == 3).all()
    for dt in (torch.float32, torch.bfloat16):
        x = _rand((5, 30, 50), 21, dt)
        out = torch.zeros(30, 5, 50, dtype=dt, device="cuda").transpose(0, 1)
        assert torch.equal(orthogonalize(x, out=out), orthogonalize(x))
        out.copy_(x)
        assert torch.equal(orthogonalize(out, out=out), orthogonalize(x))
        pair = torch.zeros(30, 110, dtype=dt, device="cuda")
        pair[:, :50] = x[0]
        orthogonalize(pair[:, :50], out=pair[:, 60:])
        assert torch.equal(pair[:, 60:], orthogonalize(x[0])) and torch.equal(pair[:, :50], x[0]) and not pair[:, 50:60].any()
        with pytest.raises(ValueError):
            orthogonalize(pair[:, :50], out=pair[:, 49:99])
        with pytest.raises(ValueError):
            orthogonalize(x, out=torch.zeros(32, 90, dtype=dt, device="cuda").as_strided((5, 30, 50), (40, 90, 1)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_gradient_beside_its_logits(dtype):
    from mcts_q_amd.policyloss import policy_loss, preference_loss
    V = 700
    buf = torch.full((4, 6, 2 * V + 9), 7.0, dtype=dtype, device="cuda")
    z, out = buf[:, :, :V], buf[:, :, V + 9:]
    z.copy_(_rand(z.shape, 1, dtype))
    a = torch.randint(0, V, (4, 6), device="cuda")
    adv, ref = torch.ones(4, 6, device="cuda"), torch.zeros(4, device="cuda")
    keep = z.clone()
    for f in (lambda **k: policy_loss(z, a, None, adv, **k), lambda **k: preference_loss(z, a, ref, **k)):
        want = f()["dlogits"]
        f(out=out)
        assert torch.equal(z, keep) and (buf[:, :, V:V + 9] == 7).all()
        assert (out.float() - want.float()).abs().max() <= 2 * torch.finfo(dtype).eps * want.float().abs().max()
        for bad in (buf[:, :, V - 1:2 * V - 1], buf[:, :, 1:V + 1], buf.view(-1)[3:3 + 24 * V].view(4, 6, V)):
            with pytest.raises(ValueError, match="out"):
                f(out=bad)
    assert torch.equal(z, keep)


def test_a_gradient_over_what_other_rows_read():
    """Weights, actions, old log-probabilities in the memory that the gradient is written to: refused by name."""
    from mcts_q_amd.policyloss import policy_loss, preference_loss
    z = _rand((4, 6, 50), 1)
    out = torch.zeros(4, 6, 50, device="cuda")
    a, f, s = torch.zeros(4, 6, dtype=torch.int64, device="cuda"), torch.zeros(4, 6, device="cuda"), torch.zeros(4, device="cuda")
    inside = out.view(-1)[100:124].view(4, 6)
    act = out.view(-1)[100:148].view(torch.int64).view(4, 6)
    vec = out.view(-1)[7:11]
    for name, call in (("old_logp", lambda: policy_loss(z, a, inside, f, out=out)),
                       ("advantages", lambda: policy_loss(z, a, f, inside, out=out)),
                       ("advantages", lambda: policy_loss(z, a, f, vec, out=out)),
                       ("ref_logp", lambda: policy_loss(z, a, f, f, ref_logp=inside, out=out)),
                       ("weight", lambda: policy_loss(z, a, f, f, weight=inside, out=out)),
                       ("actions", lambda: policy_loss(z, act, f, f, out=out)),
                       ("actions", lambda: preference_loss(z, act, s, out=out)),
                       ("ref_logp", lambda: preference_loss(z, a, vec, out=out)),
                       ("weight", lambda: preference_loss(z, a, s, weight=inside, out=out)),
                       ("pair_weight", lambda: preference_loss(z, a, s, pair_weight=vec[:2], out=out))):
        with pytest.raises(ValueError, match=name):
            call()
    assert not out.any()
