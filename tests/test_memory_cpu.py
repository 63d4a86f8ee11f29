"""Which strided tensors share memory, against the sets of their elements' addresses."""
import itertools
import random

import pytest
import torch

from mcts_q_amd._memory import overlaps_itself, share_memory, span


def _bytes(t):
    at = torch.zeros((), dtype=torch.int64)
    for s, st in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(s) * st
    first = t.data_ptr()
    return [first + t.element_size() * int(e) + k for e in at.reshape(-1) for k in range(t.element_size())]


def _check(a, b):
    sa, sb = _bytes(a), _bytes(b)
    assert share_memory(a, b) == bool(set(sa) & set(sb)) == share_memory(b, a)
    for t, s in ((a, sa), (b, sb)):
        assert overlaps_itself(t) == (len(set(s)) < len(s))
        if s:
            assert span(t) == (min(s), max(s) + 1)


def test_named_cases():
    w = torch.zeros(6, 20)
    assert share_memory(w[:, :8], w[:, 4:12]) and not share_memory(w[:, :8], w[:, 8:16])
    assert share_memory(w[2:4], w[:, 3:5]) and not share_memory(w[:3], w[3:]) and not share_memory(w, torch.zeros(6, 20))
    assert not share_memory(w[:0], w) and not overlaps_itself(w[:0])
    stack = torch.zeros(5, 3, 7).transpose(0, 1)             # rows of three matrices, in turn
    assert not overlaps_itself(stack) and not share_memory(stack[0], stack[1]) and share_memory(stack[0], stack)
    assert overlaps_itself(w[:1].expand(6, 20)) and overlaps_itself(w.as_strided((3, 5), (4, 1)))
    assert overlaps_itself(w.as_strided((2, 3, 8), (10, 20, 1), 0)) is False
    assert overlaps_itself(w.as_strided((2, 3, 11), (10, 20, 1), 0)) is True


@pytest.mark.parametrize("seed", range(30))
def test_random_views(seed):
    """Any strides, types and offsets over one small buffer; every second pair with rows of one distance."""
    rng = random.Random(seed)
    raw = torch.zeros(4096, dtype=torch.uint8)
    for trial in range(40):
        views = []
        step = rng.choice([3, 4, 7, 8, 12])
        for _ in range(2):
            dt = rng.choice([torch.float32, torch.bfloat16])
            base = raw.view(dt)
            dims = rng.choice([1, 2, 2, 3])
            shape = [rng.choice([1, 2, 3, 5]) for _ in range(dims)]
            if dims == 2 and trial % 2:
                stride = [step * 4 // base.element_size(), 1]
            else:
                stride = [rng.choice([0, 1, 2, 3, 5, 6, 10, 15, 30]) for _ in range(dims)]
                if rng.random() < 0.7:
                    stride[-1] = 1
            views.append(base.as_strided(shape, stride, rng.randrange(0, 40)))
        _check(*views)


def test_every_small_pair_of_rows():
    w = torch.zeros(64)
    rows = [w.as_strided((n, c), (ld, 1), o) for n, c, ld, o in itertools.product((1, 2, 3), (1, 2, 4), (4, 5), (0, 1, 3, 6, 13))]
    for a, b in itertools.product(rows, rows):
        _check(a, b)


def test_large_layouts_are_cheap():
    """No element is looked at: rows are, and contiguous tensors not even those."""
    big = torch.empty((1 << 16, 1 << 12), device="meta")
    assert not overlaps_itself(big) and not overlaps_itself(big[:, :100]) and overlaps_itself(big[:1].expand(5, 1 << 12))
