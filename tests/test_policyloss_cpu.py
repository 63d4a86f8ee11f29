"""The host-side checks of the policy losses' C entry points: every refused call returns < 0 with a message before
anything is launched (device pointers here are made up and never followed)."""
import ctypes

import pytest
import torch

from mcts_q_amd import MctsqError
from mcts_q_amd._lib import lib

P = 1 << 20         # stands for a device pointer


def _logp(logits=P, dtype=1, rows=12, inner=3, so=300, si=100, V=100, act=P, ab=8, w=None, out=P):
    return lib.mctsq_token_logprobs(logits, dtype, rows, inner, so, si, V, act, ab, w, out, None)


def _policy(dtype=1, rows=12, inner=3, so=300, si=100, V=100, adv=P, adv_div=1, lo=0.2, hi=0.2, kl=0.0, scale=1.0, loss=P,
            d=P, dso=300, dsi=100, ws=P, wsb=None, logits=P):
    wsb = lib.mctsq_policy_loss_workspace_bytes(rows) if wsb is None else wsb
    return lib.mctsq_policy_loss(logits, dtype, rows, inner, so, si, V, P, 8, None, None, adv, adv_div, None, lo, hi, kl, scale,
                                 loss, P, P, d, dso, dsi, ws, wsb, None)


def _pref(pairs=2, T=3, so=300, si=100, V=100, ref=P, beta=0.1, e=0.0, ws=P, wsb=None, dso=300, dsi=100):
    wsb = lib.mctsq_preference_loss_workspace_bytes(pairs, T) if wsb is None else wsb
    return lib.mctsq_preference_loss(P, 1, pairs, T, so, si, V, P, 4, ref, None, None, beta, e, 1.0, P, P, P, P, dso, dsi, ws,
                                     wsb, None)


@pytest.mark.parametrize("call,word", [
    (lambda: _logp(dtype=3), b"dtype"), (lambda: _logp(rows=-3), b"rows"), (lambda: _logp(rows=13), b"multiple"),
    (lambda: _logp(V=0), b"vocab"), (lambda: _logp(ab=2), b"4- or 8-byte"), (lambda: _logp(logits=None), b"NULL"),
    (lambda: _logp(act=None), b"NULL"), (lambda: _logp(out=None), b"NULL"), (lambda: _logp(logits=P + 1), b"aligned"),
    (lambda: _logp(so=-300), b"negative strides"), (lambda: _policy(adv=None), b"NULL"), (lambda: _policy(adv_div=0), b"adv_div"),
    (lambda: _policy(lo=-0.1), b"clip"), (lambda: _policy(hi=float("nan")), b"clip"), (lambda: _policy(kl=float("nan")), b"NaN"),
    (lambda: _policy(ws=None), b"workspace"), (lambda: _policy(wsb=8), b"workspace"), (lambda: _policy(dsi=99), b"overlap"),
    (lambda: _policy(dso=250), b"overlap"), (lambda: _policy(d=P + 1), b"aligned"), (lambda: _policy(loss=None), b"NULL"),
    (lambda: _pref(pairs=-1, wsb=1 << 20), b"out of range"), (lambda: _pref(ref=None), b"NULL"), (lambda: _pref(e=0.7), b"smoothing"),
    (lambda: _pref(beta=float("nan")), b"NaN"), (lambda: _pref(wsb=16), b"workspace"), (lambda: _pref(ws=P + 8), b"workspace"),
    (lambda: _pref(dsi=10), b"overlap")])
def test_refused_calls(call, word):
    assert call() < 0
    assert word in lib.mctsq_last_error(), lib.mctsq_last_error()


def test_workspace_queries():
    assert lib.mctsq_policy_loss_workspace_bytes(0) >= 8
    assert lib.mctsq_policy_loss_workspace_bytes(1 << 40) == 8 * 16384
    assert lib.mctsq_policy_loss_workspace_bytes(-1) < 0
    assert lib.mctsq_preference_loss_workspace_bytes(0, 0) >= 16
    assert lib.mctsq_preference_loss_workspace_bytes(1 << 20, 1 << 12) >= (1 << 33) * 20      # past 32 bits
    assert lib.mctsq_preference_loss_workspace_bytes(-1, 5) < 0


def test_no_cpu_fallback():
    from mcts_q_amd.policyloss import policy_loss, preference_loss, token_logprobs
    z, a = torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.int64)
    for f in (lambda: token_logprobs(z, a), lambda: policy_loss(z, a, None, torch.zeros(2, 3)),
              lambda: preference_loss(z, a, torch.zeros(2))):
        with pytest.raises(MctsqError):
            f()


def test_sizes_whose_products_leave_64_bits():
    """2 * 2^30 * 2^33 = 2^64 rows would count as none; 2^59 * 2^3 bytes likewise."""
    for pairs, tokens in ((1 << 30, 1 << 33), (1 << 59, 1), (1, 1 << 62)):
        assert lib.mctsq_preference_loss_workspace_bytes(pairs, tokens) < 0
        assert b"out of range" in lib.mctsq_last_error()
        assert _pref(pairs=pairs, T=tokens, wsb=1 << 20) < 0
        assert b"out of range" in lib.mctsq_last_error()
