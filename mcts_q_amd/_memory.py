"""Which bytes a strided tensor touches, for the checks that what a kernel writes is nobody else's: exact where bounding
ranges would refuse interleaved views, or pass views that cross each other's rows."""
from __future__ import annotations

import numpy as np
import torch


def span(t):
    """[first, last) byte addresses a tensor touches; empty tensors touch none."""
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride())))


def _runs(t):
    """(bytes of a contiguous run, [(count, step in bytes) ...] of the runs' starts, whether some of them coincide).
    Neighbouring dimensions that continue each other are one."""
    dims = sorted((st, s) for s, st in zip(t.shape, t.stride()) if s > 1)
    run, rest, twice = t.element_size(), [], False
    for st, s in dims:
        step = st * t.element_size()
        if step == 0:
            twice = True                                     # an expanded dimension touches nothing new
        elif step == run and not rest:
            run *= s
        elif rest and step == rest[-1][0] * rest[-1][1]:
            rest[-1] = (rest[-1][0] * s, rest[-1][1])
        else:
            rest.append((s, step))
    return run, rest, twice


def _starts(t, rest):
    at = np.array([t.data_ptr()], dtype=np.int64)
    for count, step in rest:
        at = (at[:, None] + np.arange(count, dtype=np.int64) * step).reshape(-1)
    return np.sort(at)


def overlaps_itself(t):
    """Whether two elements of t are the same memory."""
    if t.numel() == 0:
        return False
    run, rest, twice = _runs(t)
    if twice:
        return True
    reach = run                                              # rows within rows: each level clear of the one below
    for count, step in rest:
        if step < reach:
            break
        reach = (count - 1) * step + reach
    else:
        return False
    return bool((np.diff(_starts(t, rest)) < run).any())


def share_memory(a, b):
    """Whether some byte belongs to both tensors."""
    if a.numel() == 0 or b.numel() == 0 or a.device != b.device:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    (ra, da, _), (rb, db, _) = _runs(a), _runs(b)
    if not da and not db:
        return True
    if len(da) == 1 and len(db) == 1 and da[0][1] == db[0][1]:
        # rows of one distance: row j of b less row i of a lies d + (j - i) step on, and meets it from -rb + 1 to ra - 1
        (na, step), (nb, _), d = da[0], db[0], b0 - a0
        first, last = -((d + rb - 1) // step), (ra - 1 - d) // step
        return max(first, 1 - na) <= min(last, nb - 1)
    at, to = _starts(a, da), _starts(b, db)
    k = np.searchsorted(to, at + ra) - 1                     # the last run of b that starts before this one of a ends
    return bool(((k >= 0) & (to[np.maximum(k, 0)] + rb > at)).any())


def wrote(*tensors):
    """Tell autograd, and whoever prepared something from these tensors, that a kernel changed them: torch's own in-place
    operations count a version, a kernel's writes do not.  Tensors of inference mode carry none; a graph's replay counts nothing."""
    torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])
