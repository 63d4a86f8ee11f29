"""Host-side checks of the orthogonalised updates' C entry points (nothing is launched; pointers here are made up) and the
numerics of the split the kernels rest on, emulated on the CPU."""
import ctypes as C

import pytest
import torch

from mcts_q_amd import MctsqError
from mcts_q_amd._lib import MuonMatrix, lib

P = 1 << 20


def _list(*shapes, x=P, mom=P, out=P, ldx=None, ldo=None):
    return (MuonMatrix * len(shapes))(*[MuonMatrix(r, c, x, c if ldx is None else ldx, mom, out, c if ldo is None else ldo)
                                        for r, c in shapes])


def _step(m, n=None, dt=0, lr=0.1, mu=0.9, wd=0.0, eps=1e-7, adjust=1, ws=P, wsb=1 << 40):
    return lib.mctsq_muon_step(m, len(m) if n is None else n, dt, lr, mu, 1, wd, eps, adjust, ws, wsb, None)


def _orth(m, dt=0, eps=1e-7, ws=P, wsb=1 << 40):
    return lib.mctsq_orthogonalize(m, len(m), dt, eps, ws, wsb, None)


NAN = float("nan")


@pytest.mark.parametrize("call,word", [
    (lambda: _step(_list((0, 4))), b"sides"), (lambda: _step(_list((4, 65537))), b"sides"), (lambda: _step(_list((4, 4)), dt=2), b"dtype"),
    (lambda: _step(_list((4, 4)), n=-1), b"list"), (lambda: _step(_list((4, 4)), lr=NAN), b"NaN"), (lambda: _step(_list((4, 4)), wd=NAN), b"NaN"),
    (lambda: _step(_list((4, 4)), mu=1.0), b"momentum"), (lambda: _step(_list((4, 4)), mu=-0.1), b"momentum"),
    (lambda: _step(_list((4, 4)), eps=0.0), b"eps"), (lambda: _step(_list((4, 4)), adjust=7), b"adjust"),
    (lambda: _step(_list((4, 4)), ws=None), b"workspace"), (lambda: _step(_list((4, 4)), ws=P + 16), b"workspace"),
    (lambda: _step(_list((4, 4)), wsb=128), b"workspace"), (lambda: _step(_list((4, 4), x=None)), b"NULL"),
    (lambda: _step(_list((4, 4), mom=None)), b"NULL"), (lambda: _step(_list((4, 4), out=None)), b"NULL"),
    (lambda: _step(_list((4, 4), ldx=3)), b"leading"), (lambda: _step(_list((4, 4), ldo=3)), b"leading"),
    (lambda: _step(_list((4, 4), x=P + 1), dt=1), b"aligned"), (lambda: _step(_list((4, 4), out=P + 2)), b"aligned"),
    (lambda: _orth(_list((4, 4))), b"momentum"), (lambda: _orth(_list((4, 4), mom=None), eps=NAN), b"eps"),
    (lambda: _orth(_list((4, 4), mom=None), dt=5), b"dtype"), (lambda: _orth(_list((4, 4), mom=None, out=None)), b"NULL"),
    (lambda: _orth(_list((4, 4), mom=None, ldo=1)), b"leading"), (lambda: _orth(_list((4, 4), mom=None, x=P + 2)), b"aligned")])
def test_refused_calls(call, word):
    assert call() < 0
    assert word in lib.mctsq_last_error(), lib.mctsq_last_error()


def test_workspace_queries():
    one = lib.mctsq_muon_workspace_bytes(_list((64, 64)), 1)
    assert one >= 2 * 2 * 6 * 64 * 64
    assert lib.mctsq_muon_workspace_bytes(None, 0) >= 256
    many = _list(*[(64, 64)] * 500)
    assert one <= lib.mctsq_muon_workspace_bytes(many, 500) < 500 * one          # groups share the space
    big = _list((65536, 65536), mom=None)
    assert lib.mctsq_orthogonalize_workspace_bytes(big, 1, 1) >= 6 * 2 * (1 << 32)
    assert lib.mctsq_orthogonalize_workspace_bytes(big, 1, 0) >= 2 * 6 * 2 * (1 << 32)


def test_no_cpu_fallback():
    from mcts_q_amd.muon import DeviceMuon, orthogonalize
    with pytest.raises(MctsqError):
        orthogonalize(torch.zeros(4, 4))
    with pytest.raises(MctsqError):
        DeviceMuon([torch.zeros(4, 4)])
    with pytest.raises(ValueError):
        DeviceMuon([])


def test_planes_stay_in_range():
    """The fixed scale 2^14 of the 16-bit planes: the quintic keeps [0, 1.21] inside itself, so X, A = X X^T and
    B = b A + c A^2 stay below the type's largest value for every input."""
    a, b, c = 3.4445, -4.7750, 2.0315
    s = torch.linspace(0, 1.21, 200001, dtype=torch.float64)
    f = a * s + b * s ** 3 + c * s ** 5
    assert f.min() >= 0 and f.max() <= 1.2051
    lam = s * s
    assert (b * lam + c * lam * lam).abs().max() * 2 ** 14 < 65504 and lam.max() * 2 ** 14 < 65504
    q = a + b * lam + c * lam * lam                     # Q; Q A; and products of up to three steps' Q at 2^14, 2^12, 2^10
    assert q.abs().max() * 2 ** 14 < 65504 and (q * lam).abs().max() * 2 ** 14 < 65504
    s1 = s[s <= 1.0]
    n = torch.ones_like(s1)
    for k in range(3):
        n = n * (a + b * s1 ** 2 + c * s1 ** 4)
        s1 = a * s1 + b * s1 ** 3 + c * s1 ** 5
        assert n.abs().max() * 2 ** (14 - 2 * k) < 65504
