"""GPU: the quintic Newton-Schulz iteration and the Muon step against their formulas in 64 bits.

Tolerances, as Frobenius norms relative to the result's.  A step rounds X, A, B and its sums once each; eight such
roundings stand for the four of them in both operands of every product.  An error made at step k grows by at most the
quintic's slope, 3.4445 at 0, per later step: 1 + 3.4445 + ... + 3.4445^4 < 200.  fp32: a rounding is 2^-23 (two planes of
11 bits, sums in fp32), so 200 * 8 * 2^-23 = 1.9e-4.  bf16: one plane, half a step of 11 bits = 2^-11; the relative growth
of an error of a singular value that counts, |s f'(s) / f(s)|, is at most 1.55 on [0.68, 1.15], four roundings in five
steps: 4 * 5 * 2^-11 * 1.55 = 1.5e-2, plus the result's own rounding 2^-8."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 200 * 8 * 2.0 ** -23, torch.bfloat16: 20 * 2.0 ** -11 * 1.55 + 2.0 ** -8}
COEF = (3.4445, -4.7750, 2.0315)


def _truth(x, eps=1e-7):
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(5):
        s = x @ x.transpose(-1, -2).contiguous()
        x = COEF[0] * x + (COEF[1] * s + COEF[2] * (s @ s)) @ x
    return x.transpose(-1, -2).contiguous() if tall else x


def _close(got, ref, tol):
    err, mag = (got.double() - ref).flatten(-2).norm(dim=-1), ref.flatten(-2).norm(dim=-1)
    assert torch.isfinite(got).all()
    assert (err <= tol * mag + 1e-300).all(), (err / mag).max().item()


def _rand(shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    *s, r, c = shape
    k = max(1, min(8, r, c))
    x = torch.randn(*s, r, k, generator=g, device="cuda") @ torch.randn(*s, k, c, generator=g, device="cuda")
    return ((x + torch.randn(*shape, generator=g, device="cuda")) * 1e-2).to(dtype)


SHAPES = [(1, 1), (1, 7), (7, 1), (5, 128), (16, 16), (33, 31), (64, 64), (65, 129), (192, 64), (128, 192), (130, 70),
          (200, 513), (777, 300), (129, 2050), (1024, 640)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_orthogonalize_shapes(shape, dtype):
    from mcts_q_amd.muon import orthogonalize
    x = _rand(shape, sum(shape), dtype)
    o = orthogonalize(x)
    assert o.shape == x.shape and o.dtype == dtype
    _close(o, _truth(x), TOL[dtype])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_large_tiles_and_many_matrices(dtype):
    """Enough 128 x 128 tiles for the large-tile form; more matrices than one launch describes."""
    from mcts_q_amd.muon import orthogonalize
    x = _rand((9, 900, 1000), 5, dtype)                       # 9 * 36 = 324 tiles on and below the diagonals
    _close(orthogonalize(x), _truth(x), TOL[dtype])
    y = _rand((75, 24, 40), 6, dtype)
    _close(orthogonalize(y), _truth(y), TOL[dtype])
    z = _rand((8, 1000, 900), 7, dtype)
    _close(orthogonalize(z), _truth(z), TOL[dtype])


@pytest.mark.parametrize("shape,dtype", [((1, 1024, 4096), torch.float32), ((1, 2300, 1024), torch.bfloat16),
                                         ((8, 1024, 1000), torch.float32), ((6, 1024, 1024), torch.bfloat16),
                                         ((1, 577, 4100), torch.float32), ((2, 3000, 513), torch.float32)],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v)[6:])
def test_every_plan_and_tile(shape, dtype):
    """Sizes at which several steps are made at once on the smaller side, and the largest tiles, with ragged ends."""
    from mcts_q_amd.muon import orthogonalize
    x = _rand(shape, sum(shape), dtype)
    _close(orthogonalize(x), _truth(x), TOL[dtype])


@pytest.mark.parametrize("shape", [(3, 40000), (20000, 40), (1, 65536)])
def test_long_and_thin(shape):
    from mcts_q_amd.muon import orthogonalize
    x = _rand(shape, 13)
    _close(orthogonalize(x), _truth(x), TOL[torch.float32])


def test_a_mixed_list_of_large_and_small():
    """One step of 43 matrices (more than one launch group) from 8 x 9 to 1500 x 600, a NaN in one of them."""
    from mcts_q_amd.muon import DeviceMuon
    shapes = [(8, 9), (1500, 600), (600, 1500), (64, 64), (700, 700)] + [(32 + i, 100) for i in range(38)]
    params = [_rand(s, i) for i, s in enumerate(shapes)]
    start = [p.double() for p in params]
    grads = [_rand(s, 50 + i) for i, s in enumerate(shapes)]
    grads[3][5, 5] = float("nan")
    DeviceMuon(params, lr=0.1, momentum=0.5, adjust="none").step(grads)
    for i, (p, s, g) in enumerate(zip(params, start, grads)):
        if i == 3:
            assert p.isnan().all()
            continue
        want = s - 0.1 * _truth(g.double() * 1.5)
        assert (p.double() - want).norm() <= TOL[torch.float32] * (want - s).norm() + 2.0 ** -23 * want.norm(), i


def test_known_results():
    """Rank one: the iteration acts on the one singular value, 1.  Zero: zero.  1 x 1: the sign times the same value."""
    from mcts_q_amd.muon import orthogonalize
    f = 1.0
    for _ in range(5):
        f = COEF[0] * f + COEF[1] * f ** 3 + COEF[2] * f ** 5
    u, v = torch.randn(70, 1, device="cuda"), torch.randn(1, 150, device="cuda")
    # eps against a norm of about 100: 1e-9 of the value
    _close(orthogonalize(u @ v), f * (u.double() @ v.double()) / (u.double().norm() * v.double().norm()), TOL[torch.float32])
    one = orthogonalize(torch.tensor([[[3.0]], [[-1e-3]], [[2e20]]], device="cuda"))
    assert ((one.flatten().double().cpu() - f * torch.tensor([1.0, -1.0, 1.0])).abs() <= TOL[torch.float32] + 5e-4).all()
    for dt in (torch.float32, torch.bfloat16):
        assert not orthogonalize(torch.zeros(100, 30, dtype=dt, device="cuda")).any()
        assert not orthogonalize(torch.zeros(3, 300, 400, dtype=dt, device="cuda"), eps=1e-300).any()
        assert not orthogonalize(torch.zeros(3, 5, dtype=dt, device="cuda"), eps=1e-300).any()
    s = torch.linalg.svdvals(orthogonalize(_rand((300, 500), 3)).double())
    assert s.max() < 1.21 and s.min() > 0.3


@pytest.mark.parametrize("scale", [1e-36, 1e-12, 1.0, 1e15, 1e36])
def test_any_scale(scale):
    """From next to the smallest normal numbers to squares far beyond fp32: the norm is fp64, the planes are scaled."""
    from mcts_q_amd.muon import orthogonalize
    x = _rand((90, 140), 8) * scale
    _close(orthogonalize(x, eps=1e-300), _truth(x, eps=1e-300), TOL[torch.float32])
    y = _rand((90, 140), 8) * 1e-3
    _close(orthogonalize(y), _truth(y), TOL[torch.float32])
    rows = _rand((100, 200), 9) * torch.logspace(-6, 0, 100, device="cuda")[:, None]
    _close(orthogonalize(rows), _truth(rows), TOL[torch.float32])


def test_nan_and_infinity_stay_in_their_matrix():
    from mcts_q_amd.muon import orthogonalize
    x = _rand((4, 80, 150), 10)
    good = orthogonalize(x)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[1, 3, 5] = bad
        o = orthogonalize(y)
        assert o[1].isnan().all()
        keep = [0, 2, 3]
        assert torch.equal(o[keep], good[keep])


def test_views_in_place_and_untouched_surroundings():
    from mcts_q_amd.muon import orthogonalize
    for dt in (torch.float32, torch.bfloat16):
        buf = torch.full((3, 50, 91), 7.0, dtype=dt, device="cuda")
        view = buf[:, 2:47, 5:82]
        x = _rand((3, 45, 77), 11, dt)
        view.copy_(x)
        ref = orthogonalize(x)
        assert torch.equal(orthogonalize(view), ref)
        assert orthogonalize(view, out=view) is view and torch.equal(view, ref)
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask[:, 2:47, 5:82] = False
        assert (buf[mask] == 7).all()


def _muon64(p, g, m, lr, mu, nesterov, wd, factor):
    m = mu * m + g.double()
    u = g.double() + mu * m if nesterov else m
    return p * (1 - lr * wd) - lr * factor * _truth(u), m


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("nesterov,wd,adjust", [(True, 0.0, "spectral"), (False, 0.1, "rms"), (True, 0.05, "none")])
def test_steps(grad, nesterov, wd, adjust):
    """Three steps of a mixed list, stacks and strided views among it, in 64 bits from the same gradients."""
    from mcts_q_amd.muon import DeviceMuon
    shapes = [(192, 64), (64, 192), (3, 40, 65), (128, 128), (5, 128), (1, 9), (300, 140)]
    store = torch.zeros(300, 150, device="cuda")
    params = [_rand(s, i) for i, s in enumerate(shapes[:-1])]
    store[:, 4:144] = _rand(shapes[-1], 77)
    params.append(store[:, 4:144])
    opt = DeviceMuon(params, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=wd, adjust=adjust)
    p64, m64 = [p.double() for p in params], [torch.zeros_like(p, dtype=torch.float64) for p in params]
    moved = [torch.zeros((), device="cuda", dtype=torch.float64) for _ in params]
    for step in range(3):
        grads = [_rand(s, 100 * step + i, grad) for i, s in enumerate(shapes)]
        wide = torch.zeros(300, 160, dtype=grad, device="cuda")
        wide[:, 7:147] = grads[-1]
        opt.step(grads[:-1] + [wide[:, 7:147]])
        for i, s in enumerate(shapes):
            r, c = s[-2:]
            f = {"none": 1.0, "spectral": math.sqrt(max(1, r / c)), "rms": 0.2 * math.sqrt(max(r, c))}[adjust]
            new, m64[i] = _muon64(p64[i], grads[i], m64[i], 0.1, 0.9, nesterov, wd, f)
            moved[i] += (new - p64[i] * (1 - 0.1 * wd)).norm()
            p64[i] = new
            # the momentum: two roundings a step, at most three steps' sum
            assert ((opt.momentum_buffers[i].double() - m64[i]).abs() <= 6 * 2.0 ** -24 * (m64[i].abs() + 0.1)).all()
            err = (params[i].double() - p64[i]).norm()
            assert err <= TOL[torch.float32] * moved[i] + 3 * 2.0 ** -23 * p64[i].norm(), (i, step, float(err))
    assert not store[:, :4].any() and not store[:, 144:].any()


def test_same_bits_other_stream_and_graph():
    from mcts_q_amd.muon import DeviceMuon, orthogonalize
    x = _rand((200, 333), 20)
    first = orthogonalize(x)
    assert torch.equal(orthogonalize(x), first)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = orthogonalize(x)
    torch.cuda.synchronize()
    assert torch.equal(other, first)
    grads = [[_rand(s, 30 + 7 * k + i) for i, s in enumerate([(100, 60), (64, 64)])] for k in range(3)]
    eager = [_rand((100, 60), 1), _rand((64, 64), 2)]
    cap = [p.clone() for p in eager]
    oe, oc = DeviceMuon(eager, lr=0.1), DeviceMuon(cap, lr=0.1)
    gin = [g.clone() for g in grads[0]]
    save = [p.clone() for p in cap]
    with torch.cuda.stream(st):
        oc.step(gin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oc.step(gin)
    for p, s, m in zip(cap, save, oc.momentum_buffers):
        p.copy_(s)
        m.zero_()
    for k in range(3):
        for a, b in zip(gin, grads[k]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        oe.step(grads[k])
        assert all(torch.equal(a, b) for a, b in zip(cap, eager)), k


def test_state_and_refusals():
    from mcts_q_amd import MctsqError
    from mcts_q_amd.muon import DeviceMuon, orthogonalize
    p = [torch.zeros(8, 6, device="cuda"), torch.zeros(2, 5, 7, device="cuda")]
    g = [_rand((8, 6), 1), _rand((2, 5, 7), 2)]
    opt = DeviceMuon(p)
    opt.step(g)
    sd = opt.state_dict()
    two = DeviceMuon([q.clone() for q in p])
    two.load_state_dict(sd)
    opt.step(g, lr=0.5)
    two.step(g, lr=0.5)
    assert all(torch.equal(a, b) for a, b in zip(opt.params, two.params))
    z = torch.zeros(6, 8, device="cuda")
    for bad in (lambda: orthogonalize(z.double()), lambda: orthogonalize(z.t()), lambda: orthogonalize(z[0]),
                lambda: orthogonalize(z[:0]), lambda: orthogonalize(z, out=z[:3]), lambda: orthogonalize(z, out=z.bfloat16()),
                lambda: DeviceMuon([z.bfloat16()]), lambda: DeviceMuon([z.t()]), lambda: DeviceMuon([z], adjust="x"),
                lambda: DeviceMuon([z], momentum=1.0), lambda: DeviceMuon([z], momentum_buffers=[z[:3]]),
                lambda: DeviceMuon([z[:1].expand(6, 8)]), lambda: DeviceMuon([z, z]), lambda: DeviceMuon([z, z.view(12, 4)]),
                lambda: DeviceMuon([z.view(2, 3, 8), z[3:]]), lambda: orthogonalize(z[:, :4], out=z[:, 2:6]), lambda: opt.step(g[:1]), lambda: opt.step([g[0], g[1].bfloat16()]),
                lambda: opt.step([g[0].t(), g[1]]), lambda: opt.step([g[0].half(), g[1].half()]),
                lambda: opt.load_state_dict({"momentum_buffers": [z, z]})):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(MctsqError):
        orthogonalize(z, eps=0.0)


def test_shared_memory_is_refused():
    """A gradient that is the momentum would change between its two readings; one buffer for two states would mix them."""
    from mcts_q_amd.muon import DeviceMuon
    flat = torch.zeros(6 * 48, device="cuda")
    a, b, m, n, g, h = [flat[48 * i:48 * i + 48].view(6, 8) for i in range(6)]
    for bad in ([m, m], [m, a], [m, flat[120:168].view(6, 8)]):
        with pytest.raises(ValueError):
            DeviceMuon([a, b], momentum_buffers=bad)
    opt = DeviceMuon([a, b], momentum_buffers=[m, n])
    for bad in ([m, h], [g, n], [a, h], [g, a], [flat[72:120].view(6, 8), h], [flat[168:216].view(6, 8), h]):
        with pytest.raises(ValueError):
            opt.step(bad)
    assert not flat.any()
    g.copy_(_rand((6, 8), 1))
    opt.step([g, g])                                        # read only: one gradient for two matrices is fine
    assert torch.equal(a, b) and a.any() and not h.any()
    wide = torch.zeros(6, 20, device="cuda")
    strided = DeviceMuon([wide[:, :8]])
    with pytest.raises(ValueError):
        strided.step([wide[:, :8]])
    wide[:, 8:16] = g
    strided.step([wide[:, 8:16]])                           # interleaved rows share nothing
    assert torch.equal(wide[:, :8], a) and torch.equal(wide[:, 8:16], g) and not wide[:, 16:].any()
