"""page_plan_hip against the plan made request by request: tables, ring, slots and positions, all whole numbers and all equal."""
import random

import pytest
import torch

import paged_oracle as oracle
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def make(seed, B, page, max_pages, pool_extra, new_hi, released, short_ring=False, held_hi=None):
    """(lengths, new, table, ring, state, released) as lists: shuffled pages, every row holding what its length takes, the ring's free part anywhere in it."""
    rng = random.Random(seed)
    held_hi = max_pages * page if held_hi is None else held_hi
    lengths = [rng.choice((0, rng.randint(0, held_hi), rng.randint(0, min(held_hi, 2 * page)))) for _ in range(B)]
    new = [rng.choice((0, 1, 1, rng.randint(0, new_hi))) for _ in range(B)]
    held = [oracle.pages_of(n, page) for n in lengths]
    need = sum(oracle.pages_of(n + m, page) - h for n, m, h in zip(lengths, new, held))
    pool = sum(held) + need + pool_extra
    ids = list(range(pool))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-7] * (max_pages - h))
        at += h
    free = ids[at:]
    if short_ring:
        free = free[:rng.randint(0, max(0, need - 1))]
    head = rng.randrange(pool)
    ring = [-9] * pool
    for j, p in enumerate(free):
        ring[(head + j) % pool] = p
    gone = [rng.random() < 0.3 for _ in range(B)] if released else None
    return lengths, new, table, ring, (head, len(free)), gone


def call(lengths, new, table, ring, state, gone, page, tokens, inplace=False):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")       # noqa: E731
    args = [i32(lengths), i32(new), i32(table), i32(ring), i32(list(state))]
    plan = IU.page_plan_hip(*args, page, tokens, released=None if gone is None else torch.tensor(gone, device="cuda"), inplace=inplace)
    assert (plan.lengths is args[0]) == inplace and (plan.state is args[4]) == inplace
    if not inplace:
        assert args[0].tolist() == list(lengths) and args[4].tolist() == list(state)
    # a request's own slot is that of its first token
    assert plan.row_slots.tolist() == [plan.slots.tolist()[s] if g else -1 for s, g in zip(plan.starts.tolist(), plan.granted.tolist())]
    return args[2].tolist(), args[3].tolist(), plan.lengths.tolist(), tuple(plan.state.tolist()), plan.granted.tolist(), plan.starts.tolist(), plan.positions.tolist(), plan.slots.tolist()


def check(case, page, pad=0, tokens=None, inplace=False):
    lengths, new, table, ring, state, gone = case
    tokens = sum(new) + pad if tokens is None else tokens
    got, want = call(*case, page, tokens, inplace), oracle.plan(lengths, new, table, ring, state, page, tokens, gone)
    for name, g, w in zip(("table", "ring", "lengths", "state", "granted", "starts", "positions", "slots"), got, want):
        assert g == w, name
    return got


# rows, page, entries of a row, most new tokens, padding, released: one workgroup (about a token per row, or few tokens) and two launches
SIZES = [(1, 16, 1, 1, 0, False), (1, 16, 9, 100, 3, False), (2, 1024, 3, 900, 0, True), (63, 16, 40, 1, 0, True), (64, 32, 17, 70, 11, True), (65, 64, 5, 3, 0, False),
         (300, 16, 70, 5, 100, True), (1000, 128, 3, 2, 0, True), (1024, 16, 4, 4, 0, True), (1025, 16, 4, 4, 7, True), (2500, 32, 6, 2, 0, True), (1, 16, 800, 12000, 5, False),
         (3, 256, 40, 9000, 0, True), (100, 16, 130, 2000, 777, True),
         (16, 16, 9, 120, 0, True), (17, 16, 9, 40, 0, True), (3000, 16, 4, 1, 0, True), (4096, 16, 3, 1, 64, True), (5000, 64, 3, 1, 0, True)]


@pytest.mark.parametrize("B,page,max_pages,new_hi,pad,released", SIZES)
@pytest.mark.parametrize("short", [False, True])
def test_plan(B, page, max_pages, new_hi, pad, released, short):
    for seed in range(3):
        print(f"page plan B={B} page={page} max_pages={max_pages} new={new_hi} short={short} seed={seed}", flush=True)
        got = check(make(seed, B, page, max_pages, 3, new_hi, released, short), page, pad, inplace=seed == 1)
        slots = [s for s in got[7] if s >= 0]
        assert len(set(slots)) == len(slots)


@pytest.mark.parametrize("B,new_hi", [(40, 30), (200, 100)])
def test_tokens_behind_the_last_row_are_refused(B, new_hi):
    case = make(5, B, 16, 200, 3, new_hi, True)
    total = sum(case[1])
    for tokens in (0, 1, total // 2, total - 1):
        want = oracle.plan(*case[:5], 16, tokens, case[5])
        got = call(*case, 16, tokens)
        want[5][:] = [min(s, tokens + 1) for s in want[5]]
        assert list(got) == list(want)


def test_a_row_that_is_released_and_taken_up_again():
    """The old pages go to the ring, the new ones come from its front, in one row of the table."""
    for new in (1, 16, 17, 100, 5000):
        case = ([90, 33], [new, 0], [[10, 11, 12, 13, 14, 15] + [0] * 400, [16, 17, 18] + [0] * 403], list(range(20, 420)) + [-9] * 30, (0, 400), [True, True])
        got = check(case, 16)
        assert got[1][400:409] == [10, 11, 12, 13, 14, 15, 16, 17, 18] and got[0][0][0] == 20


def test_nothing_to_do():
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    plan = IU.page_plan_hip(empty, empty, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), torch.tensor([1, 2], dtype=torch.int32, device="cuda"),
                            torch.tensor([1, 1], dtype=torch.int32, device="cuda"), 16, 3)
    assert plan.state.tolist() == [1, 1] and plan.starts.tolist() == [0] and plan.slots.tolist() == [-1] * 3 and plan.positions.tolist() == [-1] * 3
    check(([5, 0], [0, 0], [[3], [4]], [1, 2], (0, 1), None), 16)


def test_numbers_that_no_caller_should_give():
    """Negative lengths and counts are 0, a length beyond the row is a full row, a state that no ring has is an empty ring, more pages than the ring takes
    are dropped: nothing is read or written out of place."""
    got = call([-5, 1000, 20], [3, 1, -2], [[0, 1], [2, 3], [4, 5]], [6, 7, 8, 9], (3, 2), None, 16, 8)
    assert got[2] == [3, 32, 20] and got[4] == [3, 0, 0] and got[0][0] == [9, 1] and got[7] == [144, 145, 146] + [-1] * 5
    for state in ((-1, 2), (4, 1), (0, 5), (0, -1)):
        got = call([0], [1], [[5]], [6, 7, 8, 9], state, None, 16, 1)
        assert got[2] == [0] and got[4] == [0] and got[3] == (0, 0) and got[0] == [[5]] and got[7] == [-1]
    got = call([64, 64], [0, 0], [[0, 1, 2, 3], [4, 5, 6, 7]], [9, 9, 9, 9], (1, 2), [True, True], 16, 0)
    assert got[3] == (1, 4) and got[1] == [1, 9, 9, 0]
    got = call([0] * 1100, [2 ** 31 - 1] * 1100, [[0]] * 1100, [6, 7], (0, 2), None, 16, 8)
    assert got[4] == [0] * 1100 and got[5] == [0] + [9] * 1100 and got[3] == (0, 2)
