"""Orthogonalised updates on device tensors through libmctsq_hip.so: the quintic Newton-Schulz iteration on matrices
(`orthogonalize`) and the optimizer whose step it is (`DeviceMuon`).

The iteration replaces a matrix by roughly the nearest semi-orthogonal one: X = x / |x|_F, then five times
X <- 3.4445 X + (-4.7750 A + 2.0315 A^2) X with A = X X^T, evaluated to fp32 accuracy; the result of a bf16 matrix is rounded
once, at the end.  Everything is enqueued on the current stream of the tensors' device; nothing synchronises."""
from __future__ import annotations

from bisect import bisect_left
from itertools import accumulate

import torch

from ._lib import MctsqError, MuonMatrix, lib, on_device, ptr, stream_ptr
from ._memory import overlaps_itself, share_memory, span, wrote

_DTYPE = {torch.float32: 0, torch.bfloat16: 1}
_ADJUST = {"none": 0, "spectral": 1, "rms": 2}
_ALIGN = 256


def _aligned(nbytes, device):
    buf = torch.empty(nbytes + _ALIGN, dtype=torch.uint8, device=device)
    off = -buf.data_ptr() % _ALIGN
    return buf[off:off + nbytes]


def _is_matrix(t):
    """[rows, cols] or [count, rows, cols] with at least one element and contiguous rows."""
    return t.dim() in (2, 3) and t.numel() > 0 and (t.shape[-1] == 1 or t.stride(-1) == 1) \
        and (t.shape[-2] == 1 or t.stride(-2) >= t.shape[-1])


def _ld(t):
    return t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def _slices(t):
    """(data pointer) of every matrix of a stack."""
    if t.dim() == 2:
        return [t.data_ptr()]
    step = t.stride(0) * t.element_size()
    return [t.data_ptr() + i * step for i in range(t.shape[0])]


def _sharing_pair(tensors):
    """Indices of two tensors that share memory, or None."""
    spans = [span(t) for t in tensors]
    reached = []                                             # those whose end lies past the current start
    for i in sorted(range(len(tensors)), key=spans.__getitem__):
        reached = [j for j in reached if spans[j][1] > spans[i][0]]
        for j in reached:
            if share_memory(tensors[i], tensors[j]):
                return min(i, j), max(i, j)
        reached.append(i)
    return None


def orthogonalize(x, eps=1e-7, out=None):
    """The iteration on `x` [rows, cols] or each matrix of [count, rows, cols], fp32 or bf16, rows contiguous.  Returns a
    tensor of the same shape and type (`out` if given; `out` may be `x`)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise MctsqError("orthogonalize needs a tensor on the GPU: the HIP path has no CPU fallback")
    if x.dtype not in _DTYPE:
        raise ValueError(f"x: expected fp32 or bf16, got {x.dtype}")
    if not _is_matrix(x):
        raise ValueError(f"x: expected [rows, cols] or [count, rows, cols] with contiguous rows, got {tuple(x.shape)} "
                         f"with strides {x.stride()}")
    given = out is not None
    if not given:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or not _is_matrix(out) or overlaps_itself(out):
        raise ValueError(f"out: expected {tuple(x.shape)} {x.dtype} on {x.device} with contiguous rows that do not overlap")
    elif not (out.data_ptr() == x.data_ptr() and out.stride() == x.stride()) and share_memory(x, out):
        raise ValueError("out: must be x itself or share no memory with it")
    r, c = x.shape[-2:]
    src, dst = _slices(x), _slices(out)
    lx, lo = _ld(x), _ld(out)
    mats = (MuonMatrix * len(src))(*[MuonMatrix(r, c, s, lx, None, d, lo) for s, d in zip(src, dst)])
    dt = _DTYPE[x.dtype]
    with on_device(x.device):
        need = lib.check(lib.mctsq_orthogonalize_workspace_bytes(mats, len(src), dt))
        ws = _aligned(need, x.device)
        lib.check(lib.mctsq_orthogonalize(mats, len(src), dt, eps, ptr(ws), need, stream_ptr(x.device)))
    if given:
        wrote(out)
    return out


class DeviceMuon:
    """Muon over a list of fp32 weight matrices, updated in place.

        m <- momentum m + g;  u = g + momentum m (nesterov) or m
        p <- p (1 - lr weight_decay) - lr f orthogonalize(u)

    f by `adjust`: "spectral" sqrt(max(1, rows / cols)), "rms" 0.2 sqrt(max(rows, cols)), "none" 1.  A parameter is
    [rows, cols] or a stack [count, rows, cols] of matrices, rows contiguous.  Gradients are fp32 or bf16, all of one type.
    They share no memory with the parameters or the state: `momentum_buffers` (fp32, contiguous, one per parameter).  The
    workspace is kept (8 bytes an element and 16 per square of the smaller side, of the largest twenty neighbours in the list),
    so steps of one instance belong on one stream at a time (two graphs captured from one instance must
    not run at once), and an instance has to live as long as the graphs captured from it.  Parameters that move between
    steps (`p.data = ...`) are followed; a captured graph keeps the addresses it was captured with."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, eps=1e-7, adjust="spectral",
                 momentum_buffers=None):
        params = list(params)
        if not params:
            raise ValueError("params: empty")
        if adjust not in _ADJUST:
            raise ValueError(f"adjust: expected one of {sorted(_ADJUST)}, got {adjust!r}")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"momentum must lie in [0, 1), got {momentum}")
        self._check_params(params, getattr(params[0], "device", None))
        self.params, self.device = params, params[0].device
        self.lr, self.momentum, self.nesterov = float(lr), float(momentum), bool(nesterov)
        self.weight_decay, self.eps, self.adjust = float(weight_decay), float(eps), adjust
        if momentum_buffers is None:
            momentum_buffers = [torch.zeros(p.shape, dtype=torch.float32, device=p.device) for p in params]
        self.momentum_buffers = list(momentum_buffers)
        self._lay_out()
        with on_device(self.device):
            self._ws_bytes = lib.check(lib.mctsq_muon_workspace_bytes(self._mats, len(self._mats)))
            self._ws = _aligned(self._ws_bytes, self.device)
            self._ws_stream = stream_ptr(self.device)

    @staticmethod
    def _check_params(params, device):
        for i, p in enumerate(params):
            if not isinstance(p, torch.Tensor) or not p.is_cuda:
                raise MctsqError("DeviceMuon needs parameters on the GPU: the HIP path has no CPU fallback")
            if p.dtype != torch.float32 or not _is_matrix(p) or p.device != device or overlaps_itself(p):
                raise ValueError(f"params[{i}]: expected fp32 [rows, cols] or [count, rows, cols] with contiguous rows on "
                                 f"{device}, got {tuple(p.shape)} {p.dtype} with strides {p.stride()} on {p.device}")
        pair = _sharing_pair(params)
        if pair:
            raise ValueError("params[%d] and params[%d] share memory" % pair)

    def _places(self):
        """Where parameters and momentum lie; `p.data = ...` (Module.to and the like) moves them."""
        return [(t.data_ptr(), t.shape, t.stride(), t.dtype) for t in (*self.params, *self.momentum_buffers)]

    def _lay_out(self):
        """The matrices' descriptions and the ranges a step writes, of the tensors as they are now."""
        params = self.params
        for i, (p, m) in enumerate(zip(params, self.momentum_buffers, strict=True)):
            if m.shape != p.shape or m.dtype != torch.float32 or m.device != p.device or not m.is_contiguous():
                raise ValueError(f"momentum_buffers[{i}]: expected contiguous fp32 {tuple(p.shape)} on {p.device}")
        if _sharing_pair(params + self.momentum_buffers):
            raise ValueError("momentum_buffers: must share no memory with each other or the parameters")
        # what a step writes, in the order of memory: starts, and how far everything up to there reaches
        self._written = sorted(params + self.momentum_buffers, key=span)
        self._first = [span(t)[0] for t in self._written]
        self._reach = list(accumulate((span(t)[1] for t in self._written), max))
        mats, self._at = [], []
        for p, m in zip(params, self.momentum_buffers):
            self._at.append(len(mats))
            mats += [MuonMatrix(p.shape[-2], p.shape[-1], None, 0, b, a, _ld(p)) for a, b in zip(_slices(p), _slices(m))]
        self._mats = (MuonMatrix * len(mats))(*mats)
        self._placed = self._places()

    def _follow(self):
        """Parameters or momentum that have moved since the last step are written where they are now."""
        now = self._places()
        if now == self._placed:
            return
        if [p[1] for p in now] != [p[1] for p in self._placed]:
            raise ValueError("params / momentum_buffers: their shapes have changed, make a new DeviceMuon")
        self._check_params(self.params, self.device)
        self._lay_out()

    def step(self, grads, lr=None):
        """One update from `grads` (a sequence in the order of the parameters)."""
        self._follow()
        if len(grads) != len(self.params):
            raise ValueError(f"grads: expected {len(self.params)} tensors, got {len(grads)}")
        dt = grads[0].dtype
        if dt not in _DTYPE:
            raise ValueError(f"grads: expected fp32 or bf16, got {dt}")
        for i, (g, p, at) in enumerate(zip(grads, self.params, self._at)):
            if g.shape != p.shape or g.dtype != dt or g.device != self.device or not _is_matrix(g):
                raise ValueError(f"grads[{i}]: expected {tuple(p.shape)} {dt} on {self.device} with contiguous rows, got "
                                 f"{tuple(g.shape)} {g.dtype} with strides {g.stride()} on {g.device}")
            a, b = span(g)
            k = bisect_left(self._first, b)                  # what starts before the gradient's end; most reaches not as far
            if k and self._reach[k - 1] > a and any(share_memory(g, t) for t in self._written[:k]):
                raise ValueError(f"grads[{i}]: must share no memory with the parameters or the momentum")
            ld = _ld(g)
            for j, q in enumerate(_slices(g)):
                self._mats[at + j].d_x, self._mats[at + j].ldx = q, ld
        with on_device(self.device):
            if stream_ptr(self.device) != self._ws_stream and not torch.cuda.is_current_stream_capturing():
                self._ws.record_stream(torch.cuda.current_stream(self.device))       # not reused before that work is done
            lib.check(lib.mctsq_muon_step(self._mats, len(self._mats), _DTYPE[dt], self.lr if lr is None else float(lr),
                                          self.momentum, int(self.nesterov), self.weight_decay, self.eps,
                                          _ADJUST[self.adjust], ptr(self._ws), self._ws_bytes, stream_ptr(self.device)))
        wrote(*self.params, *self.momentum_buffers)

    def state_dict(self):
        return {"momentum_buffers": [m.clone() for m in self.momentum_buffers]}

    def load_state_dict(self, sd):
        for m, s in zip(self.momentum_buffers, sd["momentum_buffers"], strict=True):
            if tuple(s.shape) != tuple(m.shape):
                raise ValueError(f"momentum buffer: expected {tuple(m.shape)}, got {tuple(s.shape)}")
            m.copy_(s)
