"""The preference loss's workspace query at the ends of what 64 bits hold (nothing is launched)."""
import pytest

from mcts_q_amd._lib import lib

P = 1 << 20         # stands for a device pointer


@pytest.mark.parametrize("pairs,tokens", [(1 << 30, 1 << 31), (1 << 30, 1 << 30), (1 << 28, 1 << 30), (1 << 30, (1 << 27) + 1),
                                          (1 << 59, 1), (1, 1 << 62), (-1, 3), (3, -1)])
def test_refused(pairs, tokens):
    """More than 2^58 rows: 20 bytes each and the sequences' own leave 64 bits (2^30 x 2^30 came back as 16 bytes)."""
    assert lib.mctsq_preference_loss_workspace_bytes(pairs, tokens) < 0
    assert b"out of range" in lib.mctsq_last_error()
    assert lib.mctsq_preference_loss(P, 1, pairs, tokens, 300, 100, 100, P, 4, P, None, None, 0.1, 0.0, 1.0, P, P, P, P, 300,
                                     100, P, 1 << 62, None) < 0
    assert b"out of range" in lib.mctsq_last_error()


@pytest.mark.parametrize("pairs,tokens", [(0, 0), (0, 7), (5, 0), (1, 1), (3, 61), (1, 1 << 31), (1 << 30, 1), (1 << 30, 1 << 20),
                                          (1 << 30, 1 << 27), (1 << 26, 1 << 31)])
def test_never_smaller_than_the_rows(pairs, tokens):
    """Per row a 64-bit and three 32-bit words, per sequence one, per 64 pairs a 64-bit sum, each block rounded up to 16 bytes."""
    need = 2 * pairs * tokens * 20 + 2 * pairs * 4 + -(-pairs // 64) * 8
    got = lib.mctsq_preference_loss_workspace_bytes(pairs, tokens)
    assert max(need, 16) <= got <= need + 6 * 16
