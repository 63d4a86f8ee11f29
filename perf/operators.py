"""What a policy learns from and how its weights move: the operators that are timed, and their plain forms.

token_logprobs   log pi(a_i | row i) of one logits row per token
policy_loss      clipped policy-ratio loss with a KL term against a reference policy, and its gradient by the logits
preference_loss  paired log-ratio loss over preferred / rejected sequences, and its gradient by the logits
orthogonalize    five quintic Newton-Schulz steps: the nearest semi-orthogonal matrix, roughly, of each matrix
muon_step        momentum, orthogonalize, decay and update of a list of weight matrices in place

A case is a dict of plain values; `prepare` makes its inputs on the GPU from a seed, `run` makes one pass: in elementary
torch operations (own = False) or through the framework's entry points (own = True)."""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NS = (3.4445, -4.7750, 2.0315)      # the quintic's coefficients
STEPS = 5
EPS = 1e-7


def listed():
    return [
        # ---- log-probabilities of given tokens, no gradient: what the behaviour and reference policies are asked for
        # one token for each of 48 sequences that are being generated, a vocabulary of 32000
        dict(name="logprobs-step", op="logprobs", batch=48, tokens=1, vocab=32000, dtype="bf16", ragged=False),
        # whole sequences through the reference model, odd vocabulary and length, padded tails
        dict(name="logprobs-sequences", op="logprobs", batch=6, tokens=1023, vocab=50257, dtype="bf16", ragged=True),
        # ---- clipped policy loss and its gradient
        # the agent's learner batch over its five actions
        dict(name="policy-actions", op="policy", batch=1024, tokens=0, vocab=5, dtype="fp32", ragged=False, kl=0.0),
        # an ordinary step on odd sizes in half precision, padded tails
        dict(name="policy-odd", op="policy", batch=3, tokens=333, vocab=50257, dtype="fp16", ragged=True, kl=0.05),
        # a large step with a large vocabulary
        dict(name="policy-large", op="policy", batch=8, tokens=512, vocab=131072, dtype="bf16", ragged=True, kl=0.02),
        # ---- preference loss and its gradient
        # preferred and rejected action sequences of 25 steps, as long as the agent's price window
        dict(name="preference-actions", op="preference", pairs=64, tokens=25, vocab=5, dtype="fp32", ragged=True),
        # four pairs of short answers
        dict(name="preference-short", op="preference", pairs=4, tokens=61, vocab=32000, dtype="bf16", ragged=True),
        # eight pairs of long answers
        dict(name="preference-long", op="preference", pairs=8, tokens=511, vocab=50257, dtype="bf16", ragged=True),
        # ---- orthogonalisation of a stack of matrices
        # odd sizes, wide
        dict(name="orthogonalize-odd", op="orthogonalize", count=3, rows=777, cols=2050, dtype="bf16"),
        # the projections of several layers, one stack, in 32 bits
        dict(name="orthogonalize-stack", op="orthogonalize", count=8, rows=1024, cols=1024, dtype="fp32"),
        # ---- the update of a list of weight matrices
        # the recurrent and head matrices of the agent's gru / gru / gru network
        dict(name="muon-agent", op="muon", shapes="192x64,192x64,192x64,128x192,128x128", grad="fp32", decay=0.0),
        # the projections of one transformer layer of width 2048
        dict(name="muon-layer", op="muon", shapes="2048x2048,2048x2048,2048x2048,2048x2048,8192x2048,8192x2048,2048x8192",
             grad="bf16", decay=0.01),
    ]


def _logu(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "orthogonalize", "muon"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op in ("logprobs", "policy", "preference"):
        vocab = _logu(rng, 2, 131072)
        cap = 8 * 512 * 131072 // 4 if op != "policy" else 8 * 512 * 131072 // 2
        rows = max(2, min(8192, cap // vocab))
        n = _logu(rng, 1, rows)
        if op == "preference":
            tokens = _logu(rng, 1, max(1, n // 2))
            return dict(op=op, pairs=max(1, n // (2 * tokens)), tokens=tokens, vocab=vocab, dtype=dtype,
                        ragged=rng.random() < 0.7)
        tokens = rng.choice([0, _logu(rng, 1, n)])
        c = dict(op=op, batch=max(1, n // max(1, tokens)), tokens=tokens, vocab=vocab, dtype=dtype,
                 ragged=tokens > 1 and rng.random() < 0.7)
        if op == "policy":
            c["kl"] = rng.choice([0.0, 0.02, 0.1])
        return c
    if op == "orthogonalize":
        return dict(op=op, count=rng.randint(1, 8), rows=_logu(rng, 8, 2048), cols=_logu(rng, 8, 2048),
                    dtype=rng.choice(["bf16", "fp32"]))
    shapes = ",".join(f"{_logu(rng, 8, 2048)}x{_logu(rng, 8, 2048)}" for _ in range(rng.randint(1, 7)))
    return dict(op=op, shapes=shapes, grad=rng.choice(["bf16", "fp32"]), decay=rng.choice([0.0, 0.01]))


# ------------------------------------------------------------------------------------------------ inputs

def _lead(case):
    if case["op"] == "preference":
        return (2 * case["pairs"], case["tokens"])
    return (case["batch"], case["tokens"]) if case["tokens"] else (case["batch"],)


def _lengths_mask(lead, g):
    """Sequence lengths between a quarter and the whole, one of them full."""
    B, T = lead
    ln = torch.randint(max(1, T // 4), T + 1, (B,), generator=g, device="cuda")
    ln[0] = T
    return torch.arange(T, device="cuda")[None, :] < ln[:, None]


def _logits(lead, vocab, dtype, g):
    """Logits of a trained head: a few tokens of a row stand out, most are far below.  Rows a slab at a time."""
    n = math.prod(lead)
    z = torch.empty(n, vocab, dtype=dtype, device="cuda")
    a = torch.empty(n, dtype=torch.int64, device="cuda")
    lp = torch.empty(n, dtype=torch.float64, device="cuda")
    slab = max(1, (1 << 26) // vocab)
    for i in range(0, n, slab):
        k = min(slab, n - i)
        f = torch.randn(k, vocab, generator=g, device="cuda").mul_(2.0)
        top = torch.randint(0, vocab, (k, min(8, vocab)), generator=g, device="cuda")
        f.scatter_add_(1, top, torch.rand(top.shape, generator=g, device="cuda") * 10)
        z[i:i + k] = f
        f = z[i:i + k].float()
        noise = torch.empty_like(f).exponential_(generator=g).log_().neg_()
        a[i:i + k] = (f + noise).argmax(1)                      # an action drawn from the row's own distribution
        m = f.amax(1, keepdim=True)
        lp[i:i + k] = (f.gather(1, a[i:i + k, None]) - m).squeeze(1).double() \
            - (f - m).exp_().sum(1, dtype=torch.float64).log()
        del f, noise
    return z.view(*lead, vocab), a.view(lead), lp.view(lead)


def _gradient(shape, dtype, g):
    """A weight gradient: a few strong directions over noise."""
    *s, r, c = shape
    k = max(1, min(16, r, c))
    u = torch.randn(*s, r, k, generator=g, device="cuda")
    v = torch.randn(*s, k, c, generator=g, device="cuda") * torch.linspace(1, 0.1, k, device="cuda")[:, None]
    return ((torch.matmul(u, v) / math.sqrt(k) + torch.randn(*s, r, c, generator=g, device="cuda")) * 1e-3).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case=case)
    if op in ("logprobs", "policy", "preference"):
        lead = _lead(case)
        z, a, lp = _logits(lead, case["vocab"], DT[case["dtype"]], g)
        mask = _lengths_mask(lead, g) if case["ragged"] else torch.ones(lead, dtype=torch.bool, device="cuda")
        s["logits"], s["actions"] = z, torch.where(mask, a, -100)           # padding carries no action
        if op == "logprobs":
            s["weight"] = mask.float() if case["ragged"] else None
        elif op == "policy":
            # the behaviour policy is a few updates old, the reference policy further away; advantages are normalised
            # per sequence.  A ratio within 1e-5 of a border of the clip range is moved off it: there the gradient
            # jumps and the formula has no one value.
            d = torch.randn(lead, generator=g, device="cuda", dtype=torch.float64) * 0.15
            for border in (0.8, 1.2):
                d = torch.where((d.exp() - border).abs() < 1e-5, d + 1e-3, d)
            s["old_logp"] = (lp - d).float()
            s["ref_logp"] = (lp + torch.randn(lead, generator=g, device="cuda", dtype=torch.float64) * 0.3).float() \
                if case["kl"] else None
            s["advantages"] = torch.randn(case["batch"], generator=g, device="cuda")
            w = mask.float()
            s["weight"] = w / w.sum()
        else:
            s["weight"] = mask.float()
            noise = torch.randn(lead, generator=g, device="cuda", dtype=torch.float64) * 0.2
            s["ref_logp"] = ((lp + noise) * mask).sum(1).float()            # the reference model's sequence sums
    elif op == "orthogonalize":
        s["x"] = _gradient((case["count"], case["rows"], case["cols"]), DT[case["dtype"]], g)
    else:
        shapes = [tuple(int(n) for n in t.split("x")) for t in case["shapes"].split(",")]
        s["params"] = [torch.randn(t, generator=g, device="cuda") * 0.02 for t in shapes]
        s["grads"] = [_gradient(t, DT[case["grad"]], g) for t in shapes]
        mom = [_gradient(t, torch.float32, g) * 5 for t in shapes]
        if own:
            from mcts_q_amd.muon import DeviceMuon
            s["optimizer"] = DeviceMuon(s["params"], lr=0.02, momentum=0.95, weight_decay=case["decay"])
            for b, m in zip(s["optimizer"].momentum_buffers, mom):
                b.copy_(m)
        else:
            s["momentum"] = mom
    return s


# ------------------------------------------------------------------------------------------------ one pass

def _logp_plain(z, actions, live):
    """log pi(a) per row in 64 bits (a ratio next to the clip border decides the gradient) and the row's log-sum-exp."""
    f = z.float()
    m = f.amax(-1, keepdim=True)
    lse = m.double() + (f - m).exp().sum(-1, keepdim=True, dtype=torch.float64).log()
    za = f.gather(-1, torch.where(live, actions, 0)[..., None])
    return torch.where(live, (za.double() - lse).squeeze(-1), 0.0), lse


def _dlogits_plain(z, actions, live, lse, coef):
    """coef * (one_hot(action) - softmax(row)), 0 in rows that carry no weight."""
    coef = torch.where(live, coef, 0.0).float()[..., None]
    p = (z.float() - lse.float()).exp()
    d = p * -coef
    d.scatter_add_(-1, torch.where(live, actions, 0)[..., None], coef)
    return d.to(z.dtype)


def _quintic_plain(x):
    a, b, c = NS
    wide = x.shape[-2] <= x.shape[-1]
    x = x.float()
    x = x if wide else x.transpose(-1, -2).contiguous()
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + EPS).float()
    for _ in range(STEPS):
        s = torch.matmul(x, x.transpose(-1, -2))
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    return x if wide else x.transpose(-1, -2)


def run(s):
    case = s["case"]
    op = case["op"]
    if op == "logprobs":
        if own:
            from mcts_q_amd.policyloss import token_logprobs
            return token_logprobs(s["logits"], s["actions"], weight=s["weight"])
        live = s["weight"] != 0 if s["weight"] is not None else torch.ones_like(s["actions"], dtype=torch.bool)
        return _logp_plain(s["logits"], s["actions"], live)[0].float()
    if op == "policy":
        if own:
            from mcts_q_amd.policyloss import policy_loss
            r = policy_loss(s["logits"], s["actions"], s["old_logp"], s["advantages"], ref_logp=s["ref_logp"],
                            weight=s["weight"], clip_low=0.2, clip_high=0.2, kl_coef=case["kl"])
            return [r["loss"], r["logp"], r["kl"], r["dlogits"]]
        w, z = s["weight"], s["logits"]
        live = w != 0
        logp, lse = _logp_plain(z, s["actions"], live)
        adv = s["advantages"].double()
        adv = adv[:, None] if logp.dim() == 2 else adv
        ratio = (logp - s["old_logp"].double()).exp()
        un, cl = ratio * adv, ratio.clamp(0.8, 1.2) * adv
        loss, coef, kl = -torch.minimum(un, cl), torch.where(un <= cl, -un, 0.0), torch.zeros_like(logp)
        if s["ref_logp"] is not None:
            d = s["ref_logp"].double() - logp
            kl = torch.expm1(d) - d
            loss, coef = loss + case["kl"] * kl, coef - case["kl"] * torch.expm1(d)
        kl = torch.where(live, kl, 0.0)
        total = torch.where(live, w * loss, 0.0).sum()
        return [total.float().reshape(1), logp.float(), kl.float(), _dlogits_plain(z, s["actions"], live, lse, w * coef)]
    if op == "preference":
        if own:
            from mcts_q_amd.policyloss import preference_loss
            r = preference_loss(s["logits"], s["actions"], s["ref_logp"], weight=s["weight"], beta=0.1,
                                label_smoothing=0.05)
            return [r["loss"], r["seq_logp"], r["margin"], r["dlogits"]]
        w, z = s["weight"], s["logits"]
        live = w != 0
        logp, lse = _logp_plain(z, s["actions"], live)
        seq = (w * logp).sum(1)
        P = case["pairs"]
        lr = seq - s["ref_logp"].double()
        margin = 0.1 * (lr[:P] - lr[P:])
        up, down = torch.log1p((-margin.abs()).exp()) + (-margin).clamp(min=0), \
            torch.log1p((-margin.abs()).exp()) + margin.clamp(min=0)
        loss = (0.95 * up + 0.05 * down).sum() / P
        dm = (0.05 - 1.0 / (1.0 + margin.exp())) * (0.1 / P)
        coef = w * torch.cat([dm, -dm])[:, None]
        return [loss.float().reshape(1), seq.float(), margin.float(), _dlogits_plain(z, s["actions"], live, lse, coef)]
    if op == "orthogonalize":
        if own:
            from mcts_q_amd.muon import orthogonalize
            return orthogonalize(s["x"])
        return _quintic_plain(s["x"]).to(s["x"].dtype).contiguous()
    if own:
        s["optimizer"].step(s["grads"])
        return [list(s["params"]), list(s["optimizer"].momentum_buffers)]
    for p, gr, b in zip(s["params"], s["grads"], s["momentum"]):
        b.mul_(0.95).add_(gr.float())
        o = _quintic_plain(gr.float() + 0.95 * b)
        p.mul_(1.0 - 0.02 * case["decay"]).sub_(o * (0.02 * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))))
    return [list(s["params"]), list(s["momentum"])]


# ------------------------------------------------------------------------------------------------ work and truth

def _quintic_flops(r, c):
    n, m = min(r, c), max(r, c)
    return STEPS * (n * n * m + n * n * n + 2 * n * n * m)      # two products are symmetric: half of each is enough


def work(case):
    op = case["op"]
    if op in ("logprobs", "policy", "preference"):
        lead = _lead(case)
        n, es = math.prod(lead), 4 if case["dtype"] == "fp32" else 2
        data = n * case["vocab"] * es
        per_row = {"logprobs": 8 + 4 + 4, "policy": 8 + 4 * 5, "preference": 8 + 4}[op]
        return dict(bytes=data * (1 if op == "logprobs" else 2) + n * per_row,
                    flops=n * case["vocab"] * (4 if op == "logprobs" else 7))
    if op == "orthogonalize":
        r, c, k = case["rows"], case["cols"], case["count"]
        return dict(bytes=2 * k * r * c * (4 if case["dtype"] == "fp32" else 2), flops=k * _quintic_flops(r, c))
    shapes = [tuple(int(n) for n in t.split("x")) for t in case["shapes"].split(",")]
    gb = 4 if case["grad"] == "fp32" else 2
    return dict(bytes=sum(r * c * (gb + 16) for r, c in shapes), flops=sum(_quintic_flops(r, c) for r, c in shapes))


def _exact_rows(z, actions, live):
    """Row log-probability and softmax in 64 bits, one slab of rows at a time: (logp [n], function i, k -> p[i:i+k])."""
    n, V = z.shape
    slab = max(1, (1 << 25) // V)
    logp = torch.zeros(n, dtype=torch.float64, device=z.device)
    for i in range(0, n, slab):
        ls = torch.log_softmax(z[i:i + slab].double(), -1)
        idx = actions[i:i + slab].clamp(min=0)[:, None]
        logp[i:i + slab] = torch.where(live[i:i + slab], ls.gather(1, idx)[:, 0], 0.0)
    return logp, slab


def _exact_dlogits(z, actions, live, coef, slab):
    out = torch.zeros(z.shape, dtype=torch.float64, device=z.device)
    for i in range(0, z.shape[0], slab):
        d = -torch.softmax(z[i:i + slab].double(), -1)
        d[torch.arange(d.shape[0], device=d.device), actions[i:i + slab].clamp(min=0)] += 1.0
        out[i:i + slab] = torch.where(live[i:i + slab, None], d * coef[i:i + slab, None], 0.0)
    return out


def _exact_orthogonal(x):
    """The quintic acts on the singular values alone, so in 64 bits it is iterated on the small Gram side."""
    x = x.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + EPS)
    left = x.shape[-2] <= x.shape[-1]
    for _ in range(STEPS):
        xt = x.transpose(-1, -2).contiguous()
        g = x @ xt if left else xt @ x
        eye = torch.eye(g.shape[-1], dtype=g.dtype, device=g.device)
        poly = NS[0] * eye + g @ (NS[1] * eye + NS[2] * g)
        x = poly @ x if left else x @ poly
    return x


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("logprobs", "policy", "preference"):
        lead = _lead(case)
        z, a = s["logits"].reshape(-1, case["vocab"]), s["actions"].reshape(-1)
        w = s["weight"].reshape(-1).double() if s["weight"] is not None else torch.ones_like(a, dtype=torch.float64)
        live = w != 0
        logp, slab = _exact_rows(z, a, live)
        if op == "logprobs":
            return logp.view(lead)
        if op == "policy":
            adv = s["advantages"].double()
            adv = adv.repeat_interleave(case["tokens"]) if case["tokens"] else adv
            r = torch.exp(logp - s["old_logp"].reshape(-1).double())
            inside = torch.where(adv >= 0, r <= 1.2, r >= 0.8)
            gain = torch.where(inside, r, torch.where(adv >= 0, 1.2, 0.8)) * adv
            dl = torch.where(inside, -r * adv, 0.0)
            kl = torch.zeros_like(logp)
            if s["ref_logp"] is not None:
                e = s["ref_logp"].reshape(-1).double() - logp
                kl = torch.where(live, torch.exp(e) - e - 1.0, 0.0)
                dl = dl + case["kl"] * (1.0 - torch.exp(e))
            loss = (w * (case["kl"] * kl - gain))[live].sum().reshape(1)
            return [loss, logp.view(lead), kl.view(lead),
                    _exact_dlogits(z, a, live, w * dl, slab).view(*lead, case["vocab"])]
        P = case["pairs"]
        seq = (w * logp).view(lead).sum(1)
        h = 0.1 * ((seq[:P] - s["ref_logp"][:P].double()) - (seq[P:] - s["ref_logp"][P:].double()))
        ls = torch.nn.functional.logsigmoid
        loss = -(0.95 * ls(h) + 0.05 * ls(-h)).mean().reshape(1)
        dh = -(0.95 * torch.sigmoid(-h) - 0.05 * torch.sigmoid(h)) / P
        coef = w * (0.1 * torch.cat([dh, -dh])).repeat_interleave(case["tokens"])
        return [loss, seq, h, _exact_dlogits(z, a, live, coef, slab).view(*lead, case["vocab"])]
    if op == "orthogonalize":
        return _exact_orthogonal(s["x"])
    params, moms = [], []
    old = s["optimizer"].momentum_buffers if own else s["momentum"]
    for p, gr, b in zip(s["params"], s["grads"], old):
        b = 0.95 * b.double() + gr.double()
        o = _exact_orthogonal(gr.double() + 0.95 * b)
        scale = 0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        params.append(p.double() * (1.0 - 0.02 * case["decay"]) - scale * o)
        moms.append(b)
    return [params, moms]
