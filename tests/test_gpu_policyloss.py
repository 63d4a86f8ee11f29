"""GPU: token log-probabilities, clipped policy loss and preference loss against their formulas in 64 bits.

Tolerances.  u = 2^-24.  A row's exponentials are exp2((x - m) * log2 e) in fp32: the difference and the product round
once each and the constant is off by half a step, so an exponential is off by at most 3 |x - m| u relative, plus one step
of the instruction; a thread adds at most 128 of them in fp32 (128 u), everything after that is fp64.  With D the largest
|x - m| that still counts (exp(-D) below u / V adds nothing: D <= 40) a softmax value or a row's sum is off by
K u relative, K = 3 * 40 + 2 + 128 = 250, the log-probability by K u absolute plus its own rounding |logp| u, and a
gradient element by (K + 4) u of |c| (p + [j = a]) (its coefficient and product round) plus half a step of its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
K = 250
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _make(lead, V, dtype, seed, pad=0, shift=0, spread=3.0):
    """Logits as a view with `shift` elements before the first row and `pad` between rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = math.prod(lead)
    buf = torch.full((shift + n * (V + pad) + 8,), float("nan"), dtype=dtype, device="cuda")
    z = buf[shift:shift + n * (V + pad)].view(n, V + pad)[:, :V]
    z.copy_(torch.randn(n, V, generator=g, device="cuda") * spread)
    z = z.as_strided((*lead, V), ((lead[1] * (V + pad), V + pad, 1) if len(lead) == 2 else (V + pad, 1)), shift)
    a = torch.randint(0, V, lead, generator=g, device="cuda")
    return z, a, g


def _logp64(z, a):
    ls = torch.log_softmax(z.double(), -1)
    return ls.gather(-1, a.clamp(min=0)[..., None]).squeeze(-1)


def _check_logp(got, ref):
    assert got.dtype == torch.float32 and got.shape == ref.shape
    tol = U * (K + ref.abs())
    assert ((got.double() - ref).abs() <= tol).all(), float(((got.double() - ref).abs() / tol).max())


def _check_grad(d, z, a, coef, live):
    """d against coef * (one_hot - softmax), rows a slab at a time."""
    V = z.shape[-1]
    d, z, a, coef, live = d.reshape(-1, V), z.reshape(-1, V), a.reshape(-1), coef.reshape(-1), live.reshape(-1)
    half, tiny = torch.finfo(d.dtype).eps / 2, torch.finfo(d.dtype).tiny * torch.finfo(d.dtype).eps / 2
    for i in range(0, d.shape[0], max(1, (1 << 24) // V)):
        s = slice(i, i + max(1, (1 << 24) // V))
        p = torch.softmax(z[s].double(), -1)
        one = torch.zeros_like(p).scatter_(1, a[s].clamp(min=0)[:, None], 1.0)
        ref = torch.where(live[s, None], coef[s, None] * (one - p), 0.0)
        bound = torch.where(live[s, None], coef[s, None].abs() * (p + one), 0.0) * ((K + 4) * U) + half * ref.abs() + tiny
        err = (d[s].double() - ref).abs()
        assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())
        assert not d[s][~live[s]].any()


def _policy64(z, a, old, adv, ref, w, lo, hi, kl, scale):
    """loss, logp, k and d loss / d logp per row, by the formulas, with autograd on the row's log-probability."""
    logp = _logp64(z, a).detach().requires_grad_(True)
    live = w != 0
    r = (logp - old.double()).exp() if old is not None else (logp - logp.detach()).exp()
    A = adv.double() if adv.shape == logp.shape else adv.double()[:, None].expand(logp.shape)
    l = -torch.minimum(r * A, r.clamp(1 - lo, 1 + hi) * A)
    k = torch.zeros_like(l)
    if ref is not None:
        d = ref.double() - logp
        k = d.exp() - d - 1
        l = l + kl * k
    loss = scale * (torch.where(live, w.double() * l, 0.0)).sum()
    loss.backward()
    return loss.detach(), torch.where(live, logp.detach(), 0.0), torch.where(live, k.detach(), 0.0), logp.grad, live, \
        float((scale * w.double() * l.detach())[live].abs().sum())


def _off_border(logp, d, lo, hi):
    """Ratios at least 1e-4 off the borders, where the gradient jumps."""
    for b in (1 - lo, 1 + hi):
        d = torch.where((d.exp() - b).abs() < 1e-4, d + 1e-3, d)
    return (logp - d).float()


SIZES = [(1,), (2,), (5,), (16,), (17,), (32,), (33,), (64,), (255,), (256,), (257,), (1000,), (2031,), (4097,), (8185,),
         (8200,), (32000,), (50257,), (65521,), (70001,), (131072,)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [s[0] for s in SIZES])
def test_policy_loss_every_row_width(V, dtype):
    from mcts_q_amd.policyloss import policy_loss, token_logprobs
    n = 70 if V <= 256 else 5
    z, a, g = _make((n,), V, DT[dtype], seed=V, pad=V % 3, shift=V % 5)
    w = torch.rand(n, generator=g, device="cuda")
    w[1] = 0.0
    logp = _logp64(z, a)
    old = _off_border(logp, torch.randn(n, generator=g, device="cuda").double() * 0.3, 0.2, 0.3)
    ref = (logp + torch.randn(n, generator=g, device="cuda") * 0.5).float()
    adv = torch.randn(n, generator=g, device="cuda")
    r = policy_loss(z, a, old, adv, ref_logp=ref, weight=w, clip_low=0.2, clip_high=0.3, kl_coef=0.1, loss_scale=1.7)
    loss, lp, k, coef, live, mag = _policy64(z, a, old, adv, ref, w, 0.2, 0.3, 0.1, 1.7)
    _check_logp(r["logp"], lp)
    # k = e^d - d - 1: an error e of d = ref - logp moves it by |e^d - 1| e; ratio and k carry the log-probability's K u
    d = torch.where(live, ref.double() - lp, 0.0)
    assert ((r["kl"].double() - k).abs() <= K * U * (d.exp() - 1).abs() + 4 * U * (k + d.abs())).all()
    # every log-probability moves the loss by its coefficient (twice: r and k move as well) times K u
    e = 4 * K * U * mag + 2 * K * U * float(coef.abs().sum()) + 2 * U * float(loss.abs())
    assert abs(float(r["loss"]) - float(loss)) <= e
    # the coefficient itself moves with the log-probability: |d c / d logp| <= |c| + w (|A| r + kl e^d)
    move = K * U * 1.7 * w.double() * ((lp - old.double()).exp() * adv.double().abs() + 0.1 * d.exp())
    _check_grad_with(r["dlogits"], z, a, coef, live, move)
    assert torch.equal(token_logprobs(z, a, weight=w), r["logp"])


def _check_grad_with(d, z, a, coef, live, move):
    """_check_grad with a further absolute uncertainty `move` of each row's coefficient."""
    V = z.shape[-1]
    half, tiny = torch.finfo(d.dtype).eps / 2, torch.finfo(d.dtype).tiny * torch.finfo(d.dtype).eps / 2
    p = torch.softmax(z.double(), -1)
    one = torch.zeros_like(p).scatter_(-1, a.clamp(min=0)[..., None], 1.0)
    m = live[..., None]
    ref = torch.where(m, coef[..., None] * (one - p), 0.0)
    c = torch.where(live, coef.abs() * ((K + 4) * U) + move, 0.0)[..., None]
    bound = torch.where(m, c * (p + one), 0.0) + half * ref.abs() + tiny
    err = (d.double() - ref).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())
    assert not d[~live].any()


@pytest.mark.parametrize("dtype,V", [("fp32", 5), ("bf16", 100), ("fp16", 1001), ("bf16", 9001)])
def test_padding_rows_are_never_read(dtype, V):
    """NaN, infinities and impossible actions in padding rows; a sequence without any row; in place and apart."""
    from mcts_q_amd.policyloss import policy_loss
    B, T = 4, 7
    z, a, g = _make((B, T), V, DT[dtype], seed=3)
    w = torch.ones(B, T, device="cuda")
    w[0, 3:] = 0
    w[2] = 0                                                    # nothing left
    z[0, 3] = float("nan"); z[0, 4] = float("inf"); z[0, 5] = float("-inf"); z[2] = float("nan")
    a[0, 3:] = -100; a[2] = 10 ** 12
    old = torch.zeros(B, T, device="cuda")
    clean = torch.where(w[..., None] != 0, z, torch.zeros((), dtype=z.dtype, device="cuda"))
    old = _off_border(_logp64(clean, a.clamp(0, V - 1)), torch.randn(B, T, generator=g, device="cuda").double() * .2, .2, .2)
    old[0, 3:] = float("nan")
    adv = torch.randn(B, generator=g, device="cuda")            # one per sequence
    r = policy_loss(z, a, old, adv, weight=w)
    old_c = torch.where(w != 0, old, 0.0)
    loss, lp, k, coef, live, mag = _policy64(clean, a.clamp(0, V - 1), old_c, adv, None, w, 0.2, 0.2, 0.0, 1.0)
    _check_logp(r["logp"], lp)
    assert abs(float(r["loss"]) - float(loss)) <= 4 * K * U * mag
    move = torch.where(live, K * U * (lp - old_c.double()).exp() * adv.double().abs()[:, None], 0.0)
    _check_grad_with(r["dlogits"], clean, a.clamp(0, V - 1), torch.where(live, coef, 0.0), live, move)
    assert not r["kl"].any()
    zi = z.clone()
    r2 = policy_loss(zi, a, old, adv, weight=w, out=zi)         # the gradient over the logits
    assert r2["dlogits"] is zi and torch.equal(zi, r["dlogits"]) and torch.equal(r2["logp"], r["logp"])
    w.zero_()
    r = policy_loss(z, a, old, adv, weight=w)
    assert float(r["loss"]) == 0 and not r["dlogits"].any() and not r["logp"].any()


@pytest.mark.parametrize("dtype,V", [("fp32", 7), ("bf16", 200), ("bf16", 3001), ("fp32", 40000)])
def test_impossible_actions_are_loud_and_stay_in_their_row(dtype, V):
    from mcts_q_amd.policyloss import policy_loss
    z, a, g = _make((6,), V, DT[dtype], seed=4)
    adv = torch.ones(6, device="cuda")
    good = policy_loss(z, a, None, adv)
    for bad in (-1, V, 2 ** 40):
        b = a.clone()
        b[2] = bad
        r = policy_loss(z, b, None, adv)
        assert math.isnan(float(r["loss"])) and r["dlogits"][2].isnan().all() and r["logp"][2].isnan()
        keep = [0, 1, 3, 4, 5]
        assert torch.equal(r["dlogits"][keep], good["dlogits"][keep]) and torch.equal(r["logp"][keep], good["logp"][keep])


@pytest.mark.parametrize("dtype,V", [("fp32", 6), ("bf16", 130), ("fp16", 1500), ("fp32", 5000), ("bf16", 66000)])
def test_masked_vocabulary(dtype, V):
    """Entries at -inf and at the type's lowest value have probability 0 and gradient 0; rows of one live entry; a row of
    the lowest value only is uniform; a row of -inf only is NaN."""
    from mcts_q_amd.policyloss import policy_loss
    z, a, g = _make((6,), V, DT[dtype], seed=5, spread=2.0)
    lowest = torch.finfo(DT[dtype]).min
    keep = torch.rand(6, V, generator=g, device="cuda") < 0.3
    keep.scatter_(1, a[:, None], True)
    z[0].masked_fill_(~keep[0], float("-inf"))
    z[1].masked_fill_(~keep[1], lowest)
    z[2] = float("-inf"); z[2, a[2]] = 1.5
    z[3] = lowest
    z[5] = float("-inf")
    adv = torch.ones(6, device="cuda")
    r = policy_loss(z, a, None, adv)
    assert r["logp"][5].isnan() and r["dlogits"][5].isnan().all() and math.isnan(float(r["loss"]))
    s = slice(0, 5)
    _check_logp(r["logp"][s], _logp64(z[s], a[s]))
    assert float(r["logp"][2]) == 0.0 and not r["dlogits"][2].any()
    _check_grad(r["dlogits"][s], z[s], a[s], torch.full((5,), -1.0, device="cuda", dtype=torch.float64),
                torch.ones(5, dtype=torch.bool, device="cuda"))
    assert not r["dlogits"][0][~keep[0]].any() and not r["dlogits"][1][~keep[1]].any()


def test_slices_strides_and_index_types():
    """logits[:, :-1] of a padded buffer as it is, int32 actions, an `out` of other strides and alignment."""
    from mcts_q_amd.policyloss import policy_loss
    g = torch.Generator(device="cuda").manual_seed(6)
    B, T, V = 3, 9, 1003
    full = torch.randn(B, T + 1, V + 5, generator=g, device="cuda").to(torch.bfloat16)
    z = full[:, :-1, 1:V + 1]
    a = torch.randint(0, V, (B, T), generator=g, device="cuda")
    adv = torch.randn(B, T, generator=g, device="cuda")
    ref = policy_loss(z.contiguous(), a, None, adv)
    got = policy_loss(z, a.int(), None, adv)
    store = torch.full((T, B, V + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    out = store[:, :, 3:].transpose(0, 1)
    to = policy_loss(z, a, None, adv, out=out)
    for r in (got, to):
        assert torch.equal(r["loss"], ref["loss"]) and torch.equal(r["logp"], ref["logp"])
        # another alignment hands a row's elements to other threads: sums in fp32 in another order
        assert (r["dlogits"].float() - ref["dlogits"].float()).abs().max() <= 2.0 ** -8 * ref["dlogits"].float().abs().max()
    assert (store[:, :, :3] == 7).all()
    same = full.clone()
    zz = same[:, :-1, 1:V + 1]
    policy_loss(zz, a, None, adv, out=zz)                       # in place, through the view
    assert torch.equal(zz, got["dlogits"])
    assert torch.equal(same[:, -1], full[:, -1]) and torch.equal(same[:, :, 0], full[:, :, 0]) \
        and torch.equal(same[:, :, V + 1:], full[:, :, V + 1:])


def test_offsets_past_32_bits():
    """Rows more than 2^32 bytes and 2^31 elements from the first."""
    from mcts_q_amd.policyloss import token_logprobs
    V = 8192
    buf = torch.empty((1 << 31) + 3 * V, dtype=torch.bfloat16, device="cuda")
    z = buf.as_strided((3, V), ((1 << 30) + 8, 1))
    g = torch.Generator(device="cuda").manual_seed(7)
    z.copy_(torch.randn(3, V, generator=g, device="cuda"))
    a = torch.tensor([0, 17, V - 1], device="cuda")
    _check_logp(token_logprobs(z, a), _logp64(z, a))


@pytest.mark.parametrize("P,T,V,dtype", [(1, 1, 2, "fp32"), (64, 25, 5, "fp32"), (65, 3, 7, "bf16"), (200, 2, 9, "fp16"), (3, 1, 300, "bf16"), (2, 37, 1031, "fp16"),
                                         (2, 5, 33001, "bf16"), (1, 300, 17, "bf16"), (2, 3, 131072, "bf16")])
@pytest.mark.parametrize("smooth", [0.0, 0.1])
def test_preference_loss(P, T, V, dtype, smooth):
    from mcts_q_amd.policyloss import preference_loss
    z, a, g = _make((2 * P, T), V, DT[dtype], seed=P * T + V, pad=1)
    w = (torch.rand(2 * P, T, generator=g, device="cuda") < 0.8).float()
    w[:, 0] = 1
    w[2 * P - 1] = 0                                            # a rejected sequence without any row
    u = torch.rand(P, generator=g, device="cuda") + 0.5
    ref = (torch.where(w != 0, _logp64(z, a), 0.0).sum(1) + torch.randn(2 * P, generator=g, device="cuda")).float()
    r = preference_loss(z, a, ref, weight=w, beta=0.3, label_smoothing=smooth, pair_weight=u, loss_scale=0.5)
    logp = _logp64(z, a).requires_grad_(True)
    S = (w.double() * logp).sum(1)
    h = 0.3 * ((S[:P] - ref[:P].double()) - (S[P:] - ref[P:].double()))
    ls = torch.nn.functional.logsigmoid
    loss = 0.5 * (u.double() * (-(1 - smooth) * ls(h) - smooth * ls(-h))).sum()
    loss.backward()
    loss, h, S = loss.detach(), h.detach(), S.detach()
    eS = T * K * U                                              # error of a sequence's sum
    assert ((r["seq_logp"].double() - S).abs() <= eS + U * S.abs()).all()
    assert ((r["margin"].double() - h).abs() <= 0.6 * eS + U * h.abs()).all()
    assert abs(float(r["loss"]) - float(loss)) <= 0.5 * float(u.sum()) * 0.6 * eS + U * float(loss)
    # |d coefficient / d h| <= 1/4 of its scale
    move = torch.cat([u, u]).double()[:, None] * 0.5 * 0.3 * w * 0.25 * 0.6 * eS
    _check_grad_with(r["dlogits"], z, a, logp.grad, w != 0, move)
    zi = z.clone(memory_format=torch.preserve_format)
    r2 = preference_loss(zi, a, ref, weight=w, beta=0.3, label_smoothing=smooth, pair_weight=u, loss_scale=0.5, out=zi)
    # the copy's rows have another stride, so another alignment and another order of the fp32 sums: each side is within
    # its bound above of the formula, the two within twice that of each other
    assert ((r2["margin"] - r["margin"]).double().abs() <= 2 * (0.6 * eS + U * h.abs())).all()
    assert abs(float(r2["loss"]) - float(r["loss"])) <= 2 * (0.5 * float(u.sum()) * 0.6 * eS + U * float(loss))
    assert (zi.float() - r["dlogits"].float()).abs().max() <= 2 * torch.finfo(DT[dtype]).eps * r["dlogits"].float().abs().max()


def test_preference_padding_pairs():
    """A pair of weight 0: rows not read whatever they hold, outputs 0; extreme margins stay finite."""
    from mcts_q_amd.policyloss import preference_loss
    P, T, V = 4, 6, 700
    z, a, g = _make((2 * P, T), V, torch.bfloat16, seed=9)
    z[1] = float("nan"); z[P + 1] = float("inf"); a[1] = -100
    ref = torch.zeros(2 * P, device="cuda")
    ref[1] = float("nan")
    ref[2], ref[3] = 1e6, -1e6
    u = torch.tensor([1.0, 0.0, 1.0, 1.0], device="cuda")
    r = preference_loss(z, a, ref, pair_weight=u)
    assert torch.isfinite(r["loss"]).all() and torch.isfinite(r["dlogits"]).all() and torch.isfinite(r["margin"]).all()
    assert not r["dlogits"][1].any() and not r["dlogits"][P + 1].any() and float(r["margin"][1]) == 0
    assert not r["dlogits"][3].any()                            # h = +1e5: the loss is flat
    none = preference_loss(z, a, ref, pair_weight=torch.zeros(P, device="cuda"))
    assert float(none["loss"]) == 0 and not none["dlogits"].any()


def test_preference_weights_and_impossible_tokens():
    """Fractional and negative row weights enter the sums; a rejected sequence that holds a token of probability 0 is as
    good as told apart (loss 0), a preferred one is an infinite loss with a finite gradient."""
    from mcts_q_amd.policyloss import preference_loss
    P, T, V = 3, 4, 40
    z, a, g = _make((2 * P, T), V, torch.float32, seed=21)
    w = torch.randn(2 * P, T, generator=g, device="cuda")
    ref = torch.randn(2 * P, generator=g, device="cuda")
    r = preference_loss(z, a, ref, weight=w, beta=0.3)
    logp = _logp64(z, a).requires_grad_(True)
    S = (w.double() * logp).sum(1)
    h = 0.3 * ((S[:P] - ref[:P].double()) - (S[P:] - ref[P:].double()))
    loss = -torch.nn.functional.logsigmoid(h).mean()
    loss.backward()
    eS = float(w.abs().sum(1).max()) * K * U
    assert ((r["seq_logp"].double() - S).abs() <= eS + U * S.abs()).all()
    assert abs(float(r["loss"]) - float(loss.detach())) <= 0.6 * eS + U * float(loss.detach())
    _check_grad_with(r["dlogits"], z, a, logp.grad, w != 0, w.double().abs() * 0.3 / P * 0.25 * 0.6 * eS)
    z[P + 1, 2, a[P + 1, 2]] = float("-inf")
    r = preference_loss(z, a, ref, beta=0.3)
    assert float(r["margin"][1]) == math.inf and torch.isfinite(r["loss"]).all() and not r["dlogits"][1].any()
    assert not r["dlogits"][P + 1].any()
    z[0, 1, a[0, 1]] = float("-inf")
    r = preference_loss(z, a, ref, beta=0.3)
    assert float(r["margin"][0]) == -math.inf and float(r["loss"]) == math.inf and torch.isfinite(r["dlogits"]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [5, 200, 700, 4000, 32000, 81298])
def test_single_rows_that_are_all_but_equal(dtype, V):
    """One pair of one token each: the margin is a small difference of two log-probabilities.  Of calls of few rows an
    exponential is exp2 of an argument whose rounding is made good, so it is off by the instruction's step, 2 u; everything
    after it is fp64.  A term meets at most five of them: its own, two where a lane's maximum moves (three sweeps take 81298
    elements), the join of the lanes, the join of the waves: 10 u.  x - m rounds by |x - m| u, in fp32 by at most 40 u (a
    term further below counts for nothing); of 16-bit logits it is exact but for |x| < 2^-10, a few in 10^4 elements whose
    terms are less than a tenth of the mean: far below u.  The margin rounds once."""
    from mcts_q_amd.policyloss import preference_loss
    bound = (50 if dtype == torch.float32 else 10) * U
    for seed in range(8):
        z, a, g = _make((2, 1), V, dtype, seed=seed)
        logp = _logp64(z, a)[:, 0]
        ref = logp.float() + torch.tensor([1e-3, 0.0], device="cuda")
        h = 0.1 * ((logp[0] - ref[0].double()) - (logp[1] - ref[1].double()))
        got = preference_loss(z, a, ref, beta=0.1, grad=False)["margin"].double()
        assert abs(float(got - h)) <= 0.1 * 2 * bound + U * abs(float(h)), (seed, float(got), float(h))


def test_gradients_against_differences():
    """Central differences of the reported loss along random directions of fp32 logits: step s, the loss changes by
    s <g, v> with an error of s^2 (third derivatives of O(1)) and of the loss's own K u / s."""
    from mcts_q_amd.policyloss import policy_loss, preference_loss
    g = torch.Generator(device="cuda").manual_seed(11)
    B, T, V = 4, 6, 50
    z = torch.randn(B, T, V, generator=g, device="cuda")
    a = torch.randint(0, V, (B, T), generator=g, device="cuda")
    lp = _logp64(z, a)
    old = (lp + 0.05 * torch.randn(B, T, generator=g, device="cuda")).float()       # well inside the clip range
    ref = (lp + 0.3 * torch.randn(B, T, generator=g, device="cuda")).float()
    adv = torch.randn(B, T, generator=g, device="cuda")
    fs = [lambda x: policy_loss(x, a, old, adv, ref_logp=ref, kl_coef=0.2, loss_scale=1 / 24),
          lambda x: preference_loss(x, a, ref.sum(1), beta=0.2, label_smoothing=0.1)]
    s = 2.0 ** -7
    for f in fs:
        d = f(z)["dlogits"].double()
        for _ in range(4):
            v = torch.randn(z.shape, generator=g, device="cuda")
            v /= v.norm()
            fd = (f(z + s * v)["loss"].double() - f(z - s * v)["loss"].double()) / (2 * s)
            # fp32 rounding of z + s v moves the point by up to 4 u per element, of the loss by K u of its terms
            assert abs(float(fd) - float((d * v).sum())) <= s * s + 4 * K * U / s


def test_same_bits_other_stream_and_graph():
    """The same inputs give the same bits; on another stream; captured once and replayed with eager work between."""
    from mcts_q_amd.policyloss import policy_loss, preference_loss, token_logprobs
    g = torch.Generator(device="cuda").manual_seed(12)
    z = torch.randn(6, 11, 5003, generator=g, device="cuda").to(torch.bfloat16)
    a = torch.randint(0, 5003, (6, 11), generator=g, device="cuda")
    old = (_logp64(z, a) + 0.1).float()
    adv = torch.randn(6, 11, generator=g, device="cuda")
    ref = torch.randn(6, generator=g, device="cuda")

    def all_three(z):
        p, q = policy_loss(z, a, old, adv), preference_loss(z, a, ref)
        return [p["loss"], p["logp"], p["dlogits"], q["loss"], q["margin"], q["dlogits"], token_logprobs(z, a)]

    first = all_three(z)
    assert all(torch.equal(x, y) for x, y in zip(first, all_three(z)))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = all_three(z)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(x, y) for x, y in zip(first, other))
    zs = z.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        all_three(zs)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cap = all_three(zs)
    for i in range(3):
        zs.copy_(z.roll(i, 0))
        graph.replay()
        torch.cuda.synchronize()
        want = all_three(zs)
        assert all(torch.equal(x, y) for x, y in zip(cap, want)), i


def test_empty_batches():
    from mcts_q_amd.policyloss import policy_loss, preference_loss, token_logprobs
    e = lambda *s: torch.empty(*s, device="cuda")
    i = lambda *s: torch.empty(*s, dtype=torch.int64, device="cuda")
    assert token_logprobs(e(0, 9), i(0)).shape == (0,)
    r = policy_loss(e(2, 0, 9), i(2, 0), None, e(2, 0))
    assert float(r["loss"]) == 0 and r["dlogits"].shape == (2, 0, 9)
    r = preference_loss(e(0, 3, 9), i(0, 3), e(0))
    assert float(r["loss"]) == 0 and r["margin"].shape == (0,)
    r = preference_loss(e(2, 0, 9), i(2, 0), torch.zeros(2, device="cuda"), loss_scale=1.0)    # two empty answers
    assert abs(float(r["loss"]) - math.log(2.0)) <= 2 * U and float(r["margin"]) == 0


def test_refusals():
    from mcts_q_amd import MctsqError
    from mcts_q_amd.policyloss import policy_loss, preference_loss, token_logprobs
    z = torch.zeros(4, 6, 10, device="cuda")
    a = torch.zeros(4, 6, dtype=torch.int64, device="cuda")
    adv, f = torch.zeros(4, 6, device="cuda"), torch.zeros(4, 6, device="cuda")
    bad = [lambda: token_logprobs(z.double(), a), lambda: token_logprobs(z.transpose(1, 2), a[:, :1].expand(4, 10).contiguous()),
           lambda: token_logprobs(z, a.float()), lambda: token_logprobs(z, a[:, :5]), lambda: token_logprobs(z, a.cpu()),
           lambda: token_logprobs(z[0, 0], a[0, 0]), lambda: token_logprobs(z, a, weight=f.double()),
           lambda: policy_loss(z, a, f[:, :3], adv), lambda: policy_loss(z, a, None, adv.half()),
           lambda: policy_loss(z, a, None, None),
           lambda: policy_loss(z, a, None, adv, ref_logp=f.t()), lambda: policy_loss(z, a, None, adv, out=z[:, :5]),
           lambda: policy_loss(z, a, None, adv, out=z.bfloat16()), lambda: policy_loss(z, a, None, adv, grad=False, out=z),
           lambda: policy_loss(z[:, :, :9], a, None, adv, out=z[:, :, 1:]),     # overlaps without being the same
           lambda: preference_loss(z[:3], a[:3], f[:3, 0].contiguous()), lambda: preference_loss(z, a, f[:, 0]),
           lambda: preference_loss(z, a, None), lambda: preference_loss(z[0], a[0], f[0])]
    for i, b in enumerate(bad):
        with pytest.raises(ValueError):
            b()
            pytest.fail(f"call {i} was accepted")
    for b in (lambda: token_logprobs(z.cpu(), a.cpu()), lambda: policy_loss(z, a, None, adv, clip_low=-0.1),
              lambda: preference_loss(z, a, f[:, 0].contiguous(), label_smoothing=0.6),
              lambda: policy_loss(z, a, None, adv, out=z[:1].expand(4, 6, 10))):
        with pytest.raises((MctsqError, ValueError)):
            b()
