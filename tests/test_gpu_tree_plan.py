"""tree_plan_hip against ancestors walked one by one: whole numbers, equal."""
import random

import pytest
import torch

import tree_oracle as oracle
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(parents, lengths, granted, starts):
    print("tree plan", len(lengths), "requests,", len(parents), "rows", flush=True)
    got = IU.tree_plan_hip(i32(parents), i32(lengths), i32(granted), i32(starts))
    positions, masks = oracle.plan(parents, lengths, granted, starts)
    assert got.positions.tolist() == positions and got.masks.tolist() == masks


def tree(n, rng, kind):
    if kind == "chain":
        return [j - 1 for j in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "roots":
        return [-1] * n
    return [-1 if j == 0 or rng.random() < 0.1 else rng.randrange(max(0, j - 5), j) for j in range(n)]


@pytest.mark.parametrize("kind", ["chain", "star", "roots", "mixed"])
@pytest.mark.parametrize("n", [1, 2, 3, 31, 32, 33, 63, 64])
def test_one_tree(kind, n):
    check(tree(n, random.Random(n), kind), [n + 7], [n], [0, n])


@pytest.mark.parametrize("B,pad", [(1, 5), (3, 0), (4, 1), (5, 3000), (300, 77), (5000, 1)])
def test_many_requests(B, pad):
    rng = random.Random(B)
    counts = [rng.choice((0, 1, 2, 7, 40, 64, 65, 130)) for _ in range(B)]
    starts = [sum(counts[:b]) for b in range(B + 1)] if B < 1000 else [0]
    if B >= 1000:
        for n in counts:
            starts.append(starts[-1] + n)
    granted = [0 if rng.random() < 0.2 else n for n in counts]
    parents = [p for n in counts for p in tree(n, rng, rng.choice(("chain", "star", "mixed")))] + [3] * pad
    check(parents, [g + rng.randrange(9000) for g in granted], granted, starts)


def test_parents_that_are_none():
    """Itself, a later one, any negative number: a root of its own."""
    check([0, -7, 2, 9, 1, 4, 2 ** 31 - 1, -2 ** 31], [8], [8], [0, 8])


def test_fewer_nodes_than_rows_and_rows_beyond_the_last():
    check([-1, 0, 1, 2, -1, 0, 1, 2, -1, 0], [2, 9, 5], [2, 4, 2], [0, 4, 8, 12])       # the third one's rows are not there
    check([-1, 0, 1], [9, 9], [0, 0], [0, 2, 2])


def test_nothing():
    empty = IU.tree_plan_hip(i32([]), i32([5]), i32([0]), i32([0, 0]))
    assert empty.positions.numel() == empty.masks.numel() == 0
    none = IU.tree_plan_hip(i32([0, 1]), i32([]), i32([]), i32([0]))
    assert none.positions.tolist() == [-1, -1] and none.masks.tolist() == [0, 0]
