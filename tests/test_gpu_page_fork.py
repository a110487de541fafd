"""page_fork_hip against a walk by hand: tables, shares, the ring and every page, equal."""
import random

import pytest
import torch

import tree_oracle as oracle
from paged_oracle import pages_of
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def on(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Cache:
    """Rows of the given lengths; rows in `together` share the whole pages that the shortest of them has."""

    def __init__(self, lengths, page=16, spare=9, layers=3, kv=2, d=64, together=(), seed=0, wide=2):
        rng = random.Random(seed)
        self.page, self.lengths = page, list(lengths)
        need = [pages_of(n, page) for n in lengths]
        pool = max(1, sum(need) + spare)
        order = rng.sample(range(pool), pool)
        self.table, at = [], 0
        for n in need:
            self.table.append(order[at:at + n] + [-5] * (max(need) + wide - n))
            at += n
        free, self.shares = order[at:], [0] * pool
        if together:
            first, common = together[0], min(lengths[b] for b in together) // page
            for b in together[1:]:
                free += self.table[b][:common]
                self.table[b][:common] = self.table[first][:common]
                for p in self.table[first][:common]:
                    self.shares[p] += 1
        head = rng.randrange(pool)
        self.ring = [-9] * pool
        for j, p in enumerate(free):
            self.ring[(head + j) % pool] = p
        self.state = (head, len(free))
        self.pages = torch.randn(2, layers, pool, kv, page, d, dtype=torch.float16, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))

    def fork(self, source, inplace=True):
        """One call, checked, after which this is the cache that it leaves."""
        print("page fork", source[:12], self.lengths[:12], self.pages.shape, flush=True)
        k, v = self.pages.clone()
        table, ring, shares, lengths, state = on(self.table), on(self.ring), on(self.shares), on(self.lengths), on(self.state)
        got = IU.page_fork_hip(on(source), lengths, table, ring, state, shares, k, v, inplace=inplace)
        want = oracle.fork(source, self.lengths, self.table, self.ring, self.state, self.shares, self.page)
        assert table.tolist() == want[0] and ring.tolist() == want[1] and got.lengths.tolist() == want[2] and tuple(got.state.tolist()) == want[3]
        assert shares.tolist() == want[4] and got.granted.tolist() == want[5]
        assert (lengths.tolist() == want[2]) if inplace else (lengths.tolist() == self.lengths and tuple(state.tolist()) == self.state)
        for t, old in ((k, self.pages[0]), (v, self.pages[1])):
            expected = old.clone()
            for to, of, n in want[6]:
                expected[:, to, :, :n] = old[:, of, :, :n]
            assert torch.equal(t, expected)
        self.table, self.ring, self.lengths, self.state, self.shares = want[:5]
        self.pages = torch.stack([k, v])
        self.whole()
        return want

    def whole(self):
        """Every page is held by shares + 1 rows, or is free once."""
        holders = [0] * len(self.ring)
        for b, n in enumerate(self.lengths):
            for p in self.table[b][:pages_of(n, self.page)]:
                holders[p] += 1
        free = [self.ring[(self.state[0] + j) % len(self.ring)] for j in range(self.state[1])]
        assert sorted(free) == [p for p, n in enumerate(holders) if n == 0] and all(self.shares[p] == max(0, n - 1) for p, n in enumerate(holders))


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 32, 100])
@pytest.mark.parametrize("page", [16, 64])
def test_one_row_into_others(length, page):
    c = Cache([length, 0, 3, 40], page=page)
    c.fork([0, 0, 0, 3], inplace=length % 2 == 0)
    c.fork([0, 1, -1, 0])
    c.fork([-1, -1, -1, -1])
    assert c.lengths == [0] * 4 and c.state[1] == len(c.ring)


def test_rows_that_change_places():
    c = Cache([37, 50, 16, 0, 5])
    c.fork([1, 2, 3, 4, 0])
    c.fork([4, 3, 2, 1, 0])
    c.fork([1, 0, 2, 3, 4])


def test_numbers_that_no_row_has_leave_the_row():
    c = Cache([20, 30, 40])
    before = [list(r) for r in c.table]
    c.fork([7, -2, 2 ** 31 - 1])
    assert c.table == before and c.lengths == [20, 30, 40]


def test_shared_pages_are_given_back_once_by_the_last():
    c = Cache([70, 80, 90, 33], together=(0, 1, 2))
    c.fork([-1, 1, -1, 3])                        # two of three holders at once
    c.fork([0, -1, 2, 1])                         # the last one, while another row takes the pages over
    c = Cache([70, 80, 90], together=(0, 1, 2))
    c.fork([-1, -1, -1])
    c = Cache([64, 64, 64], together=(0, 1, 2))
    c.fork([1, 2, 0])


def test_pages_that_run_out():
    """In order of the rows: the first that finds none, and all later ones that need one, stay; rows that need none go on."""
    c = Cache([20, 1, 2, 3, 32, 6], spare=2)
    want = c.fork([0, 0, 0, 0, -1, 4])
    assert want[5] == [1, 1, 1, 0, 1, 1] and c.lengths == [20, 20, 20, 3, 0, 32]
    c = Cache([20, 1, 32], spare=0)
    assert c.fork([0, 0, 1])[5] == [1, 0, 0] and c.lengths == [20, 1, 32]


@pytest.mark.parametrize("page,d,kv,layers", [(16, 64, 2, 3), (64, 128, 8, 2), (1024, 8, 1, 1), (32, 72, 3, 5)])
def test_many_calls_one_after_another(page, d, kv, layers):
    rng = random.Random(page)
    B = 12
    c = Cache([rng.randrange(3 * page) for _ in range(B)], page=page, d=d, kv=kv, layers=layers, spare=2 * B, together=(1, 4, 9), seed=d)
    for step in range(6):
        c.fork([rng.choice((b, b, -1, rng.randrange(B))) for b in range(B)], inplace=step % 2 == 0)


@pytest.mark.parametrize("B,longest,wide", [(300, 60, 2), (1100, 40, 0), (70, 3000, 100), (3, 70000, 5), (16, 2900, 0), (9, 3800, 10), (64, 700, 10), (30, 1500, 20), (17, 900, 60), (40, 1900, 3)])
def test_many_rows_and_wide_tables(B, longest, wide):
    rng = random.Random(B)
    c = Cache([rng.randrange(longest) for _ in range(B)], layers=1, kv=1, d=8, spare=B, together=tuple(range(0, B, 3)), wide=wide)
    c.fork([rng.choice((b, -1, rng.randrange(B))) for b in range(B)])
    c.fork([rng.choice((b, -1, rng.randrange(B))) for b in range(B)])


def test_without_layers_and_without_rows():
    c = Cache([20, 3], layers=1)
    k, v = c.pages[:, 0].clone()
    table, ring, shares = on(c.table), on(c.ring), on(c.shares)
    got = IU.page_fork_hip(on([0, 0]), on(c.lengths), table, ring, on(c.state), shares, k, v)
    new = int(table[1, 1])
    assert got.lengths.tolist() == [20, 20] and torch.equal(k[new, :, :4], c.pages[0, 0, c.table[0][1], :, :4]) and torch.equal(v[new, :, :4], c.pages[1, 0, c.table[0][1], :, :4])
    none = IU.page_fork_hip(on([]), on([]), torch.zeros(0, 4, dtype=torch.int32, device="cuda"), ring, on(c.state), shares, k, v)
    assert none.lengths.numel() == 0 and tuple(none.state.tolist()) == c.state


def test_entries_that_are_no_page_are_left_out():
    """A table with numbers outside the pool: nothing is counted, copied or given back for them."""
    c = Cache([40, 20, 9])
    c.table[0][0], c.table[0][2], c.table[2][0] = -1, len(c.ring) + 3, 2 ** 31 - 1
    k, v = c.pages.clone()
    table, ring, shares = on(c.table), on(c.ring), on(c.shares)
    got = IU.page_fork_hip(on([0, 0, -1]), on(c.lengths), table, ring, on(c.state), shares, k, v)
    assert torch.equal(k, c.pages[0]) and torch.equal(v, c.pages[1]) and got.lengths.tolist() == [40, 40, 0]
    # row 1 gave up two pages, and holds the one good whole page of row 0, whose last page was none
    assert got.state.tolist()[1] == c.state[1] - 1 + 2 and table[1, :2].tolist() == c.table[0][:2] and shares.tolist()[c.table[0][1]] == 1 and sum(shares.tolist()) == 1
