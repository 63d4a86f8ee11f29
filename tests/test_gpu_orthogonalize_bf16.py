"""GPU: orthogonalisation of bf16 matrices is the fp32 one of the same values, rounded once.

Tolerance.  bf16 -> fp32 is exact, and the iteration is off by at most TOL relative in the Frobenius norm (200 * 8 * 2^-23:
eight roundings of 2^-23 a step, each growing by at most 1 + 3.4445 + ... + 3.4445^4 < 200 on its way).  The one rounding to
bf16 then moves an element by at most half the spacing of bf16 at its place, h(x) = 2^(floor(log2 |x|) - 8).  An error e before
it leaves |got - x| <= h(x) + 2 |e|: |e| itself, and where e carries the value over a power of two, at most another |e| for
the wider spacing there.  So what is left of |got - x| beyond h(x) has a norm of at most 2 TOL |x|."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TOL = 200 * 8 * 2.0 ** -23
COEF = (3.4445, -4.7750, 2.0315)

SHAPES = [(1, 1), (1, 9), (33, 31), (5, 128), (64, 64), (128, 192), (192, 130), (40, 1000), (200, 513), (777, 300),
          (3, 777, 1030), (2, 640, 640), (1, 1024, 4096), (6, 1024, 1024)]


def _truth(x):
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    for _ in range(5):
        s = x @ x.transpose(-1, -2).contiguous()
        x = COEF[0] * x + (COEF[1] * s + COEF[2] * (s @ s)) @ x
    return x.transpose(-1, -2).contiguous() if tall else x


def _rand(shape, seed, rest):
    """Four directions carry the matrix, everything else is `rest` of them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    *s, r, c = shape
    k = min(4, r, c)
    x = torch.randn(*s, r, k, generator=g, device="cuda") @ torch.randn(*s, k, c, generator=g, device="cuda")
    return (x + rest * torch.randn(*shape, generator=g, device="cuda")).bfloat16()


@pytest.mark.parametrize("rest", [1.0, 1e-2], ids=["ordinary", "four-directions"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_rounded_once(shape, rest):
    from mcts_q_amd.muon import orthogonalize
    x = _rand(shape, sum(shape), rest)
    got = orthogonalize(x)
    assert got.dtype == torch.bfloat16
    assert torch.equal(got, orthogonalize(x.float()).bfloat16())
    ref = _truth(x)
    half = torch.exp2(torch.floor(torch.log2(ref.abs().clamp(min=2.0 ** -126))) - 8)
    rest = ((got.double() - ref).abs() - half).clamp(min=0)
    rel = rest.flatten(-2).norm(dim=-1) / ref.flatten(-2).norm(dim=-1)
    assert (rel <= 2 * TOL).all(), rel.max().item()


def test_strided_stack_in_place():
    from mcts_q_amd.muon import orthogonalize
    buf = torch.full((3, 50, 91), 7.0, dtype=torch.bfloat16, device="cuda")
    view = buf[:, 2:47, 5:82]
    x = _rand((3, 45, 77), 4, 0.1)
    view.copy_(x)
    want = orthogonalize(x.float()).bfloat16()
    assert orthogonalize(view, out=view) is view and torch.equal(view, want)
    mask = torch.ones_like(buf, dtype=torch.bool)
    mask[:, 2:47, 5:82] = False
    assert (buf[mask] == 7).all()
