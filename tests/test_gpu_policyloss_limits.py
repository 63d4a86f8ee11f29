"""GPU: the policy losses where an exponential leaves the range of 64 bits.

A ratio or a KL term of more than e^709 is infinite in 64 bits: the formula's limit is +inf, never NaN (which stands for an
action that does not exist).  Elements of such a row's gradient are c (one_hot - p) with c = -inf: -inf at the action,
+inf where p > 0, and NaN only where an infinity meets p = 0."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _rows(V, dtype, n=9):
    g = torch.Generator(device="cuda").manual_seed(V)
    z = (torch.randn(n, V, generator=g, device="cuda") * 2).to(dtype)
    a = torch.randint(0, V, (n,), generator=g, device="cuda")
    return z, a, torch.log_softmax(z.double(), -1).gather(1, a[:, None])[:, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("V", [5, 30, 200, 700, 9001])
def test_a_reference_far_above_the_policy(V, dtype):
    """d = ref - logp: e^d - d - 1 grows without a bound; past 64 bits it is +inf whatever the fraction of d / log 2 is."""
    from mcts_q_amd.policyloss import policy_loss
    z, a, lp = _rows(V, dtype)
    d = torch.tensor([0.5, 80.0, 200.0, 709.0, 720.0, 900.0, 1100.0, 5000.0, 1e30], device="cuda", dtype=torch.float64)
    ref = (lp + d).float()
    d = ref.double() - lp
    adv = torch.ones(9, device="cuda")
    k = d.exp() - d - 1
    r = policy_loss(z, a, None, adv, ref_logp=ref, kl_coef=0.1)
    assert not r["kl"].isnan().any()
    small = torch.tensor([True, True] + [False] * 7, device="cuda")
    assert (r["kl"][~small] == math.inf).all()                       # past fp32 from d = 89 on
    # d itself is off by the log-probability's error, at most 250 u: a relative error of k of that size
    assert ((r["kl"][small].double() - k[small]).abs() <= (250 * U + U) * 1.01 * (k + d + 1)[small]).all()
    assert float(r["loss"]) == math.inf
    far = d > 712
    at = r["dlogits"].gather(1, a[:, None])[:, 0]
    assert (at[far] == -math.inf).all()
    assert not (r["dlogits"][far] < 0).scatter(1, a[far][:, None], False).any()
    # the KL term only looked at: it takes no part in the loss
    r = policy_loss(z, a, None, adv, ref_logp=ref, kl_coef=0.0)
    assert float(r["loss"]) == -9.0 and torch.isfinite(r["dlogits"]).all() and (r["kl"][~small] == math.inf).all()
    plain = policy_loss(z, a, None, adv)
    assert torch.equal(plain["dlogits"], r["dlogits"])


@pytest.mark.parametrize("V", [5, 700])
def test_a_live_action_of_probability_zero(V):
    """logit -inf at the action: logp = -inf, ratio 0, and the KL term +inf under a reference that is finite."""
    from mcts_q_amd.policyloss import policy_loss
    z, a, lp = _rows(V, torch.float32)
    z[2, a[2]] = -math.inf
    old = lp.float()
    adv = torch.ones(9, device="cuda")
    r = policy_loss(z, a, old, adv)
    assert float(r["logp"][2]) == -math.inf and not r["dlogits"][2].any() and math.isfinite(float(r["loss"]))
    r = policy_loss(z, a, old, adv, ref_logp=old, kl_coef=0.1)
    assert float(r["kl"][2]) == math.inf and float(r["loss"]) == math.inf and float(r["dlogits"][2, a[2]]) == -math.inf
    assert torch.isfinite(r["dlogits"][[0, 1, 3, 4, 5, 6, 7, 8]]).all()


@pytest.mark.parametrize("V", [5, 700])
def test_an_infinite_ratio(V):
    """A behaviour policy that gave the action (next to) no probability: r = +inf.  A positive advantage is clipped, a
    negative one is an infinite loss, an advantage of 0 takes no part."""
    from mcts_q_amd.policyloss import policy_loss
    z, a, lp = _rows(V, torch.float32)
    old = lp.float()
    old[0], old[1], old[2] = -math.inf, -5000.0, -750.0
    adv = torch.zeros(9, device="cuda")
    r = policy_loss(z, a, old, adv)
    assert float(r["loss"]) == 0.0 and not r["dlogits"].any()
    adv[:3] = 2.0
    r = policy_loss(z, a, old, adv, clip_high=0.25)
    assert float(r["loss"]) == -7.5 and not r["dlogits"].any()       # 3 * 1.25 * 2, on the flat side
    adv[0] = -2.0
    r = policy_loss(z, a, old, adv)
    assert float(r["loss"]) == math.inf


@pytest.mark.parametrize("V", [5, 700])
def test_padding_pairs_with_weights_of_nothing(V):
    """Row weights 1 / length of an empty sequence are 0 / 0: in a pair of weight 0 they are not looked at."""
    from mcts_q_amd.policyloss import preference_loss
    P, T = 70, 3
    g = torch.Generator(device="cuda").manual_seed(V)
    z = torch.randn(2 * P, T, V, generator=g, device="cuda")
    a = torch.randint(0, V, (2 * P, T), generator=g, device="cuda")
    ref = torch.zeros(2 * P, device="cuda")
    w, u = torch.full((2 * P, T), 1 / 3, device="cuda"), torch.ones(P, device="cuda")
    want = preference_loss(z, a, ref, weight=w, pair_weight=u)
    for p in (1, 66):
        w[p], w[P + p], u[p] = math.nan, math.inf, 0.0
    r = preference_loss(z, a, ref, weight=w, pair_weight=u)
    gone = torch.zeros(P, dtype=torch.bool, device="cuda")
    gone[[1, 66]] = True
    assert not r["seq_logp"][gone.repeat(2)].any() and not r["margin"][gone].any() and not r["dlogits"][gone.repeat(2)].any()
    assert math.isfinite(float(r["loss"]))
    assert torch.equal(r["seq_logp"][~gone.repeat(2)], want["seq_logp"][~gone.repeat(2)])
    assert torch.equal(r["dlogits"][~gone.repeat(2)], want["dlogits"][~gone.repeat(2)])
