"""Limits at which counts and sizes of the operators for drafted trees and settings still fit what holds them, on the CPU: every refusal comes before anything is launched, and a call on no rows
launches nothing."""
from test_tree_abi import ADJUST, L, SHAPE, call  # noqa: F401


def test_texts_whose_tokens_a_count_cannot_hold(L):  # noqa: F811
    """A token's count has 31 bits: 2^31 occurrences, in the history and on a row's path, would be none."""
    adjust = lambda **c: call(L.bs_logits_adjust_f16, ADJUST, **c)        # noqa: E731
    assert adjust(width=1 << 30, drafted_width=1 << 30) == SHAPE == adjust(width=1 << 30, drafted_width=1 << 30, R=0)
    assert adjust(width=1 << 30, drafted_width=(1 << 30) - 1, R=0) == adjust(width=(1 << 30) - 1, drafted_width=1 << 30, R=0) == adjust(width=1 << 30, drafted_width=0, R=0) == 0
