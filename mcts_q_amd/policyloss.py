"""What a policy learns from, on device tensors: log-probabilities of given actions, the clipped policy-ratio loss with a
KL term, and the paired log-ratio (preference) loss, through libmctsq_hip.so.

Like DeviceLearner's TD loss these return the gradient beside the loss (there is no autograd in this package):

    r = policy_loss(head(x), actions, old_logp, advantages, weight=mask / mask.sum())
    logits.backward(r["dlogits"])          # or any other way of carrying it on

Logits are fp32, bf16 or fp16 `[N, V]` or `[B, T, V]` with contiguous rows and any row strides (a slice such as
`logits[:, :-1]` is taken as it is).  Per-row tensors have the logits' leading shape; `weight` fp32 scales a row's share of
the loss, rows of weight 0 are padding: their logits and action are never read and their outputs are exactly 0.  An action
outside [0, V) on a row that has weight turns that row's outputs and the loss to NaN.  Everything is enqueued on the
current stream of the logits' device; nothing synchronises, scratch comes from torch's allocator.
"""
from __future__ import annotations

import functools

import torch

from ._lib import MctsqError, lib, on_device, ptr, stream_ptr
from ._memory import share_memory, wrote

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@functools.lru_cache(maxsize=256)
def _policy_ws(n):
    return lib.check(lib.mctsq_policy_loss_workspace_bytes(n))


@functools.lru_cache(maxsize=256)
def _preference_ws(pairs, tokens):
    return lib.check(lib.mctsq_preference_loss_workspace_bytes(pairs, tokens))


def _rows(logits, actions, what="logits"):
    """(rows, inner, stride_outer, stride_inner, V, leading shape) after the checks every loss shares."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise MctsqError(f"{what} must be a tensor on the GPU: the HIP path has no CPU fallback")
    if logits.dtype not in _DTYPE:
        raise ValueError(f"{what}: expected fp32, bf16 or fp16, got {logits.dtype}")
    if logits.dim() not in (2, 3) or logits.shape[-1] < 1:
        raise ValueError(f"{what}: expected [N, V] or [B, T, V] with V >= 1, got {tuple(logits.shape)}")
    if logits.shape[-1] > 1 and logits.stride(-1) != 1:
        raise ValueError(f"{what}: the elements of a row must be contiguous, got strides {logits.stride()}")
    lead = logits.shape[:-1]
    if actions.shape != lead or actions.dtype not in (torch.int32, torch.int64) or not actions.is_contiguous() \
            or actions.device != logits.device:
        raise ValueError(f"actions: expected contiguous int32 or int64 {tuple(lead)} on {logits.device}, got "
                         f"{tuple(actions.shape)} {actions.dtype} on {actions.device}")
    n = lead.numel()
    if len(lead) == 1:
        return n, max(n, 1), 0, logits.stride(0), logits.shape[-1], lead
    return n, max(lead[1], 1), logits.stride(0), logits.stride(1), logits.shape[-1], lead


def _vec(name, t, shape, device):
    if t is None:
        return
    if t.shape != shape or t.dtype != torch.float32 or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name}: expected contiguous fp32 {tuple(shape)} on {device}, got {tuple(t.shape)} {t.dtype} on "
                         f"{t.device}")


def _grad_out(logits, out, **read):
    if out is None:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device \
            or (out.shape[-1] > 1 and out.stride(-1) != 1):
        raise ValueError(f"out: expected {tuple(logits.shape)} {logits.dtype} on {logits.device} with contiguous rows, got "
                         f"{tuple(out.shape)} {out.dtype} on {out.device}")
    if not (out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()) and share_memory(logits, out):
        raise ValueError("out: must be the logits themselves or share no memory with them")
    for name, t in read.items():                             # other rows still read them while this one's gradient is written
        if t is not None and share_memory(t, out):
            raise ValueError(f"out: must share no memory with {name}")
    return out


def _out_strides(out):
    return (0, out.stride(0)) if out.dim() == 2 else (out.stride(0), out.stride(1))


def token_logprobs(logits, actions, weight=None):
    """log pi(action) of every row, fp32 in the leading shape (0 where weight is 0)."""
    n, inner, so, si, V, lead = _rows(logits, actions)
    dev = logits.device
    _vec("weight", weight, lead, dev)
    logp = torch.empty(lead, dtype=torch.float32, device=dev)
    with on_device(dev):
        lib.check(lib.mctsq_token_logprobs(ptr(logits), _DTYPE[logits.dtype], n, inner, so, si, V, ptr(actions),
                                           actions.element_size(), ptr(weight), ptr(logp), stream_ptr(dev)))
    return logp


def policy_loss(logits, actions, old_logp, advantages, ref_logp=None, weight=None, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, loss_scale=1.0, grad=True, out=None):
    """loss = loss_scale * sum_i w_i (-min(r_i A_i, clip(r_i, 1 - clip_low, 1 + clip_high) A_i) + kl_coef k_i) with
    r = exp(logp - old_logp) and k = exp(ref_logp - logp) - (ref_logp - logp) - 1.

    old_logp None: on-policy, r = 1.  ref_logp None: no KL term; kl_coef 0: k is only reported.  advantages: one per row,
    or `[B]` for `[B, T, V]` logits (one per sequence).  `out`: where the gradient goes, with strides of its own; the logits
    themselves are allowed.  Returns dict(loss [1], logp, kl (k per row), dlogits (None when grad is False))."""
    n, inner, so, si, V, lead = _rows(logits, actions)
    dev = logits.device
    for name, t in (("old_logp", old_logp), ("ref_logp", ref_logp), ("weight", weight)):
        _vec(name, t, lead, dev)
    adv_div = 1
    if advantages is None:
        raise ValueError("advantages: one per row, or one per sequence, is needed")
    if len(lead) == 2 and advantages.dim() == 1:
        _vec("advantages", advantages, lead[:1], dev)
        adv_div = inner
    else:
        _vec("advantages", advantages, lead, dev)
    if not grad and out is not None:
        raise ValueError("out is given but grad is False")
    d = _grad_out(logits, out, actions=actions, old_logp=old_logp, advantages=advantages, ref_logp=ref_logp,
                  weight=weight) if grad else None
    dso, dsi = _out_strides(d) if grad else (0, 0)
    with on_device(dev):
        need = _policy_ws(n)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        loss = torch.empty(1, dtype=torch.float32, device=dev)
        logp = torch.empty(lead, dtype=torch.float32, device=dev)
        kl = torch.empty(lead, dtype=torch.float32, device=dev)
        lib.check(lib.mctsq_policy_loss(ptr(logits), _DTYPE[logits.dtype], n, inner, so, si, V, ptr(actions),
                                        actions.element_size(), ptr(old_logp), ptr(ref_logp), ptr(advantages), adv_div,
                                        ptr(weight), clip_low, clip_high, kl_coef, loss_scale, ptr(loss), ptr(logp),
                                        ptr(kl), ptr(d), dso, dsi, ptr(ws), need, stream_ptr(dev)))
    if out is not None:
        wrote(out)
    return dict(loss=loss, logp=logp, kl=kl, dlogits=d)


def preference_loss(logits, actions, ref_logp, weight=None, beta=0.1, label_smoothing=0.0, pair_weight=None,
                    loss_scale=None, grad=True, out=None):
    """Paired log-ratio loss.  logits `[2 P, T, V]`: sequence p is preferred over sequence P + p.  With the weighted sums
    S = sum_t w logp and the reference policy's sums ref_logp `[2 P]`,

        h = beta ((S_p - ref_p) - (S_{P+p} - ref_{P+p}))
        loss = loss_scale * sum_p u_p (-(1 - e) log sigmoid(h_p) - e log sigmoid(-h_p)),   e = label_smoothing

    loss_scale None: 1 / P (the mean over pairs).  pair_weight fp32 `[P]`: u; a pair of weight 0 is padding.
    Returns dict(loss [1], seq_logp [2 P], margin [P] (h), dlogits (None when grad is False))."""
    n, inner, so, si, V, lead = _rows(logits, actions)
    dev = logits.device
    if len(lead) != 2 or lead[0] % 2:
        raise ValueError(f"logits: expected [2 P, T, V], got {tuple(logits.shape)}")
    P, T = lead[0] // 2, lead[1]
    _vec("weight", weight, lead, dev)
    _vec("ref_logp", ref_logp, lead[:1], dev)
    if ref_logp is None:
        raise ValueError("ref_logp: the reference policy's sequence sums are needed")
    _vec("pair_weight", pair_weight, torch.Size((P,)), dev)
    if not grad and out is not None:
        raise ValueError("out is given but grad is False")
    if loss_scale is None:
        loss_scale = 1.0 / max(P, 1)
    d = _grad_out(logits, out, actions=actions, ref_logp=ref_logp, weight=weight, pair_weight=pair_weight) if grad else None
    dso, dsi = _out_strides(d) if grad else (0, 0)
    with on_device(dev):
        need = _preference_ws(P, T)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        loss = torch.empty(1, dtype=torch.float32, device=dev)
        seq = torch.empty(2 * P, dtype=torch.float32, device=dev)
        margin = torch.empty(P, dtype=torch.float32, device=dev)
        lib.check(lib.mctsq_preference_loss(ptr(logits), _DTYPE[logits.dtype], P, T, so, si, V, ptr(actions),
                                            actions.element_size(), ptr(ref_logp), ptr(weight), ptr(pair_weight), beta,
                                            label_smoothing, loss_scale, ptr(loss), ptr(seq), ptr(margin), ptr(d), dso,
                                            dsi, ptr(ws), need, stream_ptr(dev)))
    if out is not None:
        wrote(out)
    return dict(loss=loss, seq_logp=seq, margin=margin, dlogits=d)
