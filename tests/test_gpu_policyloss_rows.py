"""GPU: the policy losses over many rows, with and without a gradient: every kernel that large calls launch, in every type, and
workgroups that take more than one round of rows.

Tolerances, u = 2^-24.  With d_j = x_j - max of a row, an exponential's argument rounds twice (the difference, the product
with log2 e in two words): 2 |d_j| u, wherever a running maximum moves on the way, as the parts add up to d_j; every
exponential or rescaling is off by the instruction's step, 2 u, besides: one for the element, at most S = 8 sweeps of a row,
two joins; two fp32 additions come before fp64.  A row's sum, and so its log-probability, is off by
e = (2 sum_j p_j |d_j| + 2 (1 + 8 + 2) + 2) u at most, p the row's softmax.  A gradient element c (one - p): the exponential is
made with log2 e in one word (3 |d_j| u), the sum adds e, rounding of coefficient, reciprocal, products and the last addition
8 u; the coefficient itself moves by its derivative times e."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _make(n, V, dtype, pad, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.full((3 + n * (V + pad) + 8,), float("nan"), dtype=DT[dtype], device="cuda")
    z = buf[3 if pad else 0:].as_strided((n, V), (V + pad, 1))
    for s in range(0, n, 1 << 14):                            # a slab at a time: the random numbers are fp32
        k = min(n, s + (1 << 14))
        z[s:k] = (torch.randn(k - s, V, generator=g, device="cuda") * 3).to(DT[dtype])
    return z, torch.randint(0, V, (n,), generator=g, device="cuda"), g


def _slabs(n, V):
    step = max(1, (1 << 23) // V)
    return [slice(s, min(n, s + step)) for s in range(0, n, step)]


def _rows64(z, a):
    """log-probability and its bound e, per row."""
    lp, e = [], []
    for s in _slabs(*z.shape):
        x = z[s].double()
        d = x - x.max(1, keepdim=True).values
        l = torch.log_softmax(x, 1)
        lp.append(l.gather(1, a[s, None])[:, 0])
        e.append((2 * (l.exp() * d.abs()).sum(1) + 24) * U)
    return torch.cat(lp), torch.cat(e)


def _check_logp(got, lp, e, live):
    assert ((got.double() - lp).abs() <= e + U * lp.abs())[live].all(), float(((got.double() - lp).abs() / e)[live].max())
    assert not got[~live].any()


def _check_grad(dz, z, a, c, e, move, live):
    half, tiny = torch.finfo(dz.dtype).eps / 2, torch.finfo(dz.dtype).tiny * torch.finfo(dz.dtype).eps / 2
    for s in _slabs(*z.shape):
        x = z[s].double()
        d, p = (x - x.max(1, keepdim=True).values).abs(), torch.softmax(x, 1)
        one = torch.zeros_like(p).scatter_(1, a[s, None], 1.0)
        on = live[s, None]
        ref = torch.where(on, c[s, None] * (one - p), 0.0)
        bound = torch.where(on, c[s, None].abs() * (p * ((3 * d + 8) * U + e[s, None]) + 8 * U * one) + move[s, None] * (p + one), 0.0)
        err = (dz[s].double() - ref).abs()
        assert (err <= bound + half * ref.abs() + tiny).all(), float((err / (bound + half * ref.abs() + tiny)).max())
        assert not dz[s][~live[s]].any()


def _policy(n, V, dtype, pad=3, seed=0):
    from mcts_q_amd.policyloss import policy_loss, token_logprobs
    z, a, g = _make(n, V, dtype, pad, seed or n + V)
    w = torch.rand(n, generator=g, device="cuda")
    w[torch.rand(n, generator=g, device="cuda") < 0.1] = 0.0
    lp, e = _rows64(z, a)
    delta = torch.randn(n, generator=g, device="cuda").double() * 0.3
    for b in (0.8, 1.25):                                     # ratios off the borders, where the gradient jumps
        delta = torch.where((delta.exp() - b).abs() < 1e-4, delta + 1e-3, delta)
    old, ref = (lp - delta).float(), (lp + torch.randn(n, generator=g, device="cuda") * 0.5).float()
    adv, live = torch.randn(n, generator=g, device="cuda"), w != 0
    args = dict(ref_logp=ref, weight=w, clip_low=0.2, clip_high=0.25, kl_coef=0.1, loss_scale=1.7)
    got = policy_loss(z, a, old, adv, **args)
    A, W, r, k = adv.double(), 1.7 * w.double(), (lp - old.double()).exp(), ref.double() - lp
    un, cl, ek = r * A, r.clamp(0.8, 1.25) * A, k.exp()
    k = ek - k - 1
    c = W * (torch.where(un <= cl, -un, 0.0) - 0.1 * (ek - 1))
    loss = W * (-torch.minimum(un, cl) + 0.1 * k)
    _check_logp(got["logp"], lp, e, live)
    assert ((got["kl"].double() - k).abs() <= (ek - 1).abs() * e + 4 * U * (k + 1))[live].all() and not got["kl"][~live].any()
    move = W * (A.abs() * r + 0.1 * ek) * e
    bound = float((c.abs() * e + move * e).sum()) + 2 * U * abs(float(loss.sum()))
    assert abs(float(got["loss"]) - float(loss.sum())) <= bound
    _check_grad(got["dlogits"], z, a, c, e, move, live)
    # nothing but the gradient's absence changes without it; in place nothing but the place (the same alignment)
    none = policy_loss(z, a, old, adv, grad=False, **args)
    assert none["dlogits"] is None and all(torch.equal(none[k], got[k]) for k in ("logp", "kl", "loss"))
    _check_logp(token_logprobs(z, a, weight=w), lp, e, live)
    want = got["dlogits"].clone()
    over = policy_loss(z, a, old, adv, out=z, **args)
    assert torch.equal(over["logp"], got["logp"]) and torch.equal(over["loss"], got["loss"])
    # an aligned and an unaligned store hold the same values: only the rows' own alignment moves elements between threads
    assert torch.equal(z, want)


# a row's vectors: one wave, up to eight a lane; two, four waves; eight streamed; sixteen held, streamed
WIDTHS = [257, 490, 1000, 2031, 4070, 8171, 16330, 32000, 65100, 131072]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V", WIDTHS)
def test_more_rows_than_the_chip_has_compute_units(V, dtype):
    _policy(257 + V % 50, V, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,V", [(300, 5), (1024, 8), (1025, 8), (40, 30), (20, 250), (3, 490), (4, 4070), (6, 33000), (2, 131072)])
def test_fewer_rows(n, V, dtype):
    _policy(n, V, dtype)


@pytest.mark.parametrize("dtype,n,V", [("bf16", 600, 8300), ("fp16", 530, 40001), ("fp32", 520, 4500), ("fp32", 2100, 1500),
                                       ("bf16", 2100, 4300), ("fp16", 300, 4300)])
def test_log_probabilities_by_one_four_and_sixteen_waves(dtype, n, V):
    """Wide rows: many are taken by few waves each, few by sixteen."""
    from mcts_q_amd.policyloss import token_logprobs
    z, a, g = _make(n, V, dtype, 5, n)
    w = (torch.rand(n, generator=g, device="cuda") < 0.9).float()
    lp, e = _rows64(z, a)
    _check_logp(token_logprobs(z, a, weight=w), lp, e, w != 0)
    _check_logp(token_logprobs(z.contiguous(), a.int()), lp, e, torch.ones_like(w, dtype=torch.bool))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("P,T,V", [(70, 2, 300), (2, 70, 900), (2, 80, 2700), (3, 50, 9003), (1, 140, 20011), (2, 300, 33000)])
def test_preference_loss_of_many_rows(P, T, V, dtype):
    from mcts_q_amd.policyloss import preference_loss
    n = 2 * P * T
    z, a, g = _make(n, V, dtype, 2, n + V)
    w = (torch.rand(n, generator=g, device="cuda") < 0.8).float()
    w[0] = 1.0
    lp, e = _rows64(z, a)
    live = (w != 0)
    S, eS = torch.where(live, lp, 0.0).view(2 * P, T).sum(1), torch.where(live, e, 0.0).view(2 * P, T).sum(1)
    ref = (S + torch.randn(2 * P, generator=g, device="cuda")).float()
    got = preference_loss(z.as_strided((2 * P, T, V), (T * z.stride(0), z.stride(0), 1)), a.view(2 * P, T), ref,
                          weight=w.view(2 * P, T), beta=0.3, label_smoothing=0.1)
    h = 0.3 * ((S[:P] - ref[:P].double()) - (S[P:] - ref[P:].double()))
    eh = 0.3 * (eS[:P] + eS[P:])
    assert ((got["seq_logp"].double() - S).abs() <= eS + U * S.abs()).all()
    assert ((got["margin"].double() - h).abs() <= eh + U * h.abs()).all()
    ls = torch.nn.functional.logsigmoid
    loss = (-0.9 * ls(h) - 0.1 * ls(-h)).mean()
    assert abs(float(got["loss"]) - float(loss)) <= float(eh.mean()) + U * float(loss)
    c = 0.3 / P * (0.1 - torch.sigmoid(-h))
    c, move = torch.cat([c, -c]).repeat_interleave(T), (0.3 / P * 0.25 * eh).repeat(2).repeat_interleave(T)
    _check_grad(got["dlogits"].view(n, V), z, a, c, e, move, live)
    none = preference_loss(z.as_strided((2 * P, T, V), (T * z.stride(0), z.stride(0), 1)), a.view(2 * P, T), ref,
                           weight=w.view(2 * P, T), beta=0.3, label_smoothing=0.1, grad=False)
    assert none["dlogits"] is None and all(torch.equal(none[k], got[k]) for k in ("seq_logp", "margin", "loss"))


# more rows than one round of the grid takes: 16384 workgroups of 256, 64, 16, four and one row
@pytest.mark.parametrize("dtype,n,V", [("bf16", 16384 * 256 + 77, 5), ("fp32", 16384 * 64 + 77, 9), ("fp16", 16384 * 16 + 77, 33),
                                       ("bf16", 4 * 16384 + 77, 257), ("fp32", 2 * 4 * 16384 + 5, 300), ("bf16", 16384 + 77, 4200),
                                       ("fp32", 16384 + 77, 2100), ("fp16", 16384 + 300, 8300)])
def test_a_second_round_of_rows(dtype, n, V):
    _policy(n, V, dtype, pad=1)


def test_a_second_round_of_sixteen_waves():
    """The widest forms: rows of the second round behind padding rows and impossible actions of the first, whose rows and
    nobody else's become NaN."""
    from mcts_q_amd.policyloss import policy_loss
    V, n = 33000, 16384 + 260
    z = torch.randn(40, V, device="cuda").bfloat16()
    z = z.repeat(n // 40 + 1, 1)[:n]                          # row i is row i % 40
    a = torch.arange(n, device="cuda") % 40 * 811
    w = torch.ones(n, device="cuda")
    w[5:16384:7] = 0.0
    adv = torch.ones(n, device="cuda")
    r = policy_loss(z, a, None, adv, weight=w)
    one = policy_loss(z[:40], a[:40], None, adv[:40])
    live = w != 0
    assert abs(float(r["loss"]) + float(w.sum())) <= 2 * U * n
    # the small call adds its exponentials in 64 bits, the large one four at a time in 32: 2 e apart, and a bf16 step
    lp, e = _rows64(z[:40], a[:40])
    i = torch.arange(n, device="cuda") % 40
    assert ((r["logp"].double() - lp[i]).abs() <= (e + U * lp.abs())[i])[live].all() and not r["logp"][~live].any()
    for s in _slabs(n, V):
        close = (r["dlogits"][s].float() - one["dlogits"].float()[i[s]]).abs() <= 2.0 ** -7 * one["dlogits"].float().abs()[i[s]] + 1e-30
        assert close[live[s]].all() and not r["dlogits"][s][~live[s]].any()
    bad = [3, 16383, 16384 + 3, n - 1]
    a[bad] = V
    q = policy_loss(z, a, None, adv, weight=w)
    assert math.isnan(float(q["loss"])) and q["logp"][bad].isnan().all()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[bad] = False
    assert torch.equal(q["logp"][keep], r["logp"][keep])
    for s in _slabs(n, V):
        assert torch.equal(q["dlogits"][s][keep[s]], r["dlogits"][s][keep[s]]) and q["dlogits"][s][~keep[s]].isnan().all()
