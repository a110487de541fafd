"""tree_accept_hip against a walk by hand: paths, lengths, the ring, and every row of the cache, equal."""
import random

import pytest
import torch

import tree_oracle as oracle
from paged_oracle import pages_of
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def on(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


class Case:
    def __init__(self, held, counts, refused=(), page=16, layers=3, kv=2, d=64, nodes=64, pad=0, seed=0, agree=0.8, room=None, vocabulary=50):
        rng = random.Random(seed)
        B, self.page, self.nodes = len(held), page, nodes
        self.granted = [0 if b in refused else n for b, n in enumerate(counts)]
        self.lengths = [h + g for h, g in zip(held, self.granted)]
        self.starts = [sum(counts[:b]) for b in range(B + 1)]
        T = self.starts[-1] + pad
        need = [pages_of(n, page) for n in self.lengths]
        pool = sum(need) + (room if room is not None else 9)
        order = rng.sample(range(pool), pool)
        self.table, at = [], 0
        for n in need:
            self.table.append(order[at:at + n] + [-5] * (max(need) + 2 - n))
            at += n
        free = order[at:]
        head = rng.randrange(pool)
        self.ring = [-9] * pool
        for j, p in enumerate(free):
            self.ring[(head + j) % pool] = p
        self.state = (head, len(free))
        self.parents, self.tokens = [3] * T, [rng.randrange(vocabulary) for _ in range(T)]
        self.targets, self.slots = [rng.randrange(vocabulary) for _ in range(T)], [-1] * T
        for b, n in enumerate(counts):
            start = self.starts[b]
            for j in range(n):
                self.parents[start + j] = rng.randrange(max(0, j - 4), j) if j else -1
                if j and rng.random() < agree:
                    self.targets[start + self.parents[start + j]] = self.tokens[start + j]
                if self.granted[b]:
                    p = held[b] + j
                    self.slots[start + j] = self.table[b][p // page] * page + p % page
        self.pages = torch.randn(2, layers, pool, kv, page, d, dtype=torch.float16, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))

    def check(self, inplace=False):
        print("tree accept", self.granted[:8], self.lengths[:8], self.pages.shape, flush=True)
        k, v = self.pages.clone()
        lengths, state, ring, table = on(self.lengths), on(self.state), on(self.ring), on(self.table)
        got = IU.tree_accept_hip(on(self.tokens, torch.int64), on(self.parents), on(self.targets, torch.int64), on(self.slots, torch.int64), lengths, on(self.granted),
                                 on(self.starts), table, ring, state, k, v, self.nodes, inplace=inplace)
        want = oracle.accept(self.tokens, self.parents, self.targets, self.lengths, self.granted, self.starts, self.table, self.ring, self.state, self.page, self.nodes)
        assert got.lengths.tolist() == want[0] and tuple(got.state.tolist()) == want[1] and got.accepted.tolist() == want[2]
        assert got.path.tolist() == want[3] and got.token.tolist() == want[4] and ring.tolist() == want[5] and table.tolist() == self.table
        assert (lengths.tolist() == want[0] and tuple(state.tolist()) == want[1]) if inplace else (lengths.tolist() == self.lengths and tuple(state.tolist()) == self.state)
        for t, old in ((k, self.pages[0]), (v, self.pages[1])):
            assert torch.equal(t, oracle.moved(old, self.slots, self.starts, want[3], self.page))
        return want


@pytest.mark.parametrize("n", [1, 2, 3, 8, 17, 33, 63, 64])
@pytest.mark.parametrize("held", [0, 1, 15, 16, 100])
@pytest.mark.parametrize("agree", [0.0, 0.7, 1.0])
def test_one_request(n, held, agree):
    Case([held], [n], seed=n + held, agree=agree).check(inplace=n % 2 == 0)


def test_a_long_chain_moves_nothing_and_a_late_path_moves_all():
    c = Case([20], [64])
    c.parents = [j - 1 for j in range(64)]
    c.targets = c.tokens[1:] + [7]
    assert c.check()[2] == [64]
    # the odd nodes are a chain of their own behind node 0, the even ones a wrong one: every accepted row but the first two moves
    c.parents = [-1, 0, 0] + [j - 2 for j in range(3, 64)]
    c.tokens = [5] + [9 if j % 2 else 8 for j in range(1, 64)]
    c.targets = [9] * 64
    assert c.check()[3][0][:5] == [0, 1, 3, 5, 7]


@pytest.mark.parametrize("page,d,kv,layers", [(16, 64, 2, 3), (64, 128, 8, 2), (1024, 8, 1, 1), (32, 72, 3, 5), (16, 256, 1, 1)])
@pytest.mark.parametrize("inplace", [False, True])
def test_batches(page, d, kv, layers, inplace):
    rng = random.Random(page + d)
    B = 40
    Case([rng.randrange(90) for _ in range(B)], [rng.choice((0, 1, 2, 5, 16, 40, 64)) for _ in range(B)], refused=(3, 17), page=page, d=d, kv=kv, layers=layers, pad=6, seed=d).check(inplace)


def test_more_requests_than_threads():
    rng = random.Random(5)
    Case([rng.randrange(40) for _ in range(2500)], [rng.randrange(6) for _ in range(2500)], refused=range(0, 2500, 9), layers=1, kv=1, d=8, nodes=8).check()


def test_without_layers():
    c = Case([9, 30], [12, 20], layers=1)
    c.check()
    k, v = c.pages[:, 0].clone()
    ring = on(c.ring)
    got = IU.tree_accept_hip(on(c.tokens, torch.int64), on(c.parents), on(c.targets, torch.int64), on(c.slots, torch.int64), on(c.lengths), on(c.granted), on(c.starts), on(c.table),
                             ring, on(c.state), k, v)
    assert torch.equal(k, oracle.moved(c.pages[0], c.slots, c.starts, got.path.tolist(), c.page)[0])


def test_more_nodes_than_are_allowed_are_taken_back():
    want = Case([30, 30], [9, 8], nodes=8).check()
    assert want[0][0] == 30 and want[2][0] == 0 and want[4][0] == -1 and want[2][1] > 0


def test_of_children_with_one_token_the_first_counts():
    c = Case([5], [5])
    c.parents, c.tokens, c.targets = [-1, 0, 0, 1, 2], [1, 4, 4, 6, 6], [4, 6, 6, 2, 2]
    assert c.check()[3][0][:4] == [0, 1, 3, -1]


def test_tokens_are_compared_in_64_bits():
    c = Case([5], [3])
    c.parents, c.tokens, c.targets = [-1, 0, 0], [1, 2 ** 32 + 7, 7], [7, 0, 0]
    assert c.check()[3][0][:3] == [0, 2, -1]


def test_rows_without_a_slot_stay_and_a_full_ring_takes_no_more():
    c = Case([16], [40], agree=1.0)
    c.parents, c.tokens, c.targets = [-1, 0, 0] + [j - 2 for j in range(3, 40)], [5] + [9 if j % 2 else 8 for j in range(1, 40)], [9] * 40
    k, v = c.pages.clone()
    slots = list(c.slots)
    slots[3], slots[5] = -1, c.pages.shape[2] * 16                        # nodes 3 and 5, and places 3 and 5, are not there
    ring = on(list(range(len(c.ring))))
    got = IU.tree_accept_hip(on(c.tokens, torch.int64), on(c.parents), on(c.targets, torch.int64), on(slots, torch.int64), on(c.lengths), on(c.granted), on(c.starts), on(c.table),
                             ring, on((1, len(c.ring))), k, v)
    assert got.state.tolist() == [1, len(c.ring)] and ring.tolist() == list(range(len(c.ring)))
    way = got.path[0].tolist()
    want = c.pages[0].clone()
    for i, j in enumerate(way):
        if j >= 0 and i not in (3, 5) and j not in (3, 5):
            to, of = c.slots[i], c.slots[j]
            want[:, to // 16, :, to % 16] = c.pages[0][:, of // 16, :, of % 16]
    assert torch.equal(k, want) and way[:5] == [0, 1, 3, 5, 7]
