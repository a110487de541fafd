"""attention_tree_hip against attention in 64 bits, node by node.

The bound of an output o = sum_j w_j v_j: its rounding to fp16 (2^-11 |o|, or half of the smallest step, 2^-25), the weights' rounding to fp16 (2^-11 sum_j w_j |v_j|; below fp16's
full numbers, the largest weight going in as 2^15, half a step is 2^-40 of the largest), scores off by at most e (weights then by 2 e): the fp32 sum of d <= 128 products, 2^-17 sum |q k| / sqrt(d), and
the scaling of the exponent, 2^-22 |s|; and the sums' own roundings in fp32 (chains of at most 2^9 steps: 2^-15)."""
import random

import pytest
import torch

import tree_oracle as oracle
from paged_oracle import pages_of
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu
NAN = float("nan")


def on(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


class Case:
    def __init__(self, heads, kv, d, page, held, counts, nodes=None, refused=(), pad=0, seed=0, filler=NAN, max_pages=None, kind="tree", spare=2, scale=1.5):
        g, rng = torch.Generator(device="cuda").manual_seed(seed + heads + d), random.Random(seed)
        self.heads, self.kv, self.d, self.page = heads, kv, d, page
        self.nodes = nodes or max(1, max(counts))
        B = len(held)
        self.granted = [0 if b in refused else n for b, n in enumerate(counts)]
        self.lengths = [h + n for h, n in zip(held, self.granted)]
        self.starts = [sum(counts[:b]) for b in range(B + 1)]
        T = self.starts[-1] + pad
        need = [pages_of(n, page) for n in self.lengths]
        pool = sum(need) + spare
        order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
        self.rows, at = [], 0
        for n in need:
            self.rows.append(order[at:at + n])
            at += n
        wide = max_pages or max(1, max(need))
        self.table = [r + [-1] * (wide - len(r)) for r in self.rows]
        self.q = (torch.randn(T, heads * d, device="cuda", generator=g) * scale).half()
        # what nobody has written is no number
        self.kpages, self.vpages = torch.full((2, pool, kv, page, d), filler, device="cuda", dtype=torch.float16)
        for b, n in enumerate(self.lengths):
            for pages in (self.kpages, self.vpages):
                for p in range(need[b]):
                    m = min(page, n - p * page)
                    pages[self.rows[b][p], :, :m] = torch.randn(kv, m, d, device="cuda", generator=g).half()
        self.masks = [-1] * T
        for b, n in enumerate(counts):
            parents = [-1 if j == 0 else j - 1 if kind == "chain" else rng.randrange(max(0, j - 4), j) for j in range(n)]
            for j, above in enumerate(oracle.ancestors(parents)):
                mask = sum(1 << i for i in above) if kind != "any" else rng.getrandbits(64)
                self.masks[self.starts[b] + j] = mask - (1 << 64) if mask >> 63 else mask

    def args(self):
        return (self.q, self.kpages, self.vpages, on(self.table), on(self.lengths), on(self.granted), on(self.starts), on(self.masks, torch.int64), self.nodes)

    def run(self, **more):
        return IU.attention_tree_hip(*self.args(), **more)

    def check(self, out=None, bad=()):
        """bad: positions (request, position) of pages that the table does not name."""
        print("tree attention", self.heads, self.kv, self.d, self.page, self.lengths[:9], self.granted[:9], self.nodes, flush=True)
        out = self.run() if out is None else out
        worst = 0.0
        live = set()
        for b, (start, n) in enumerate(oracle.trees(self.granted, self.starts, self.q.shape[0], self.nodes)):
            if n == 0:
                continue
            length = self.lengths[b]
            keys, values = (torch.cat([t[max(r, 0)] for r in self.rows[b]], 1).transpose(0, 1)[:length] for t in (self.kpages, self.vpages))
            there = torch.ones(length, dtype=torch.bool, device="cuda")
            for request, position in bad:
                if request == b:
                    there[position] = False
            for j in range(n):
                t = start + j
                live.add(t)
                seen = there.clone()
                seen[length - n:] &= torch.tensor([bool(self.masks[t] >> i & 1) for i in range(n)], device="cuda")
                want, spread, size, lost = oracle.attend(self.q[t].view(self.heads, self.d), keys, values, seen)
                e = 2.0 ** -16 * size + 2.0 ** -20
                bound = 2.0 ** -11 * want.abs() + 2.0 ** -25 + (2.0 ** -11 + 2 * e + 2.0 ** -14) * spread + 2.0 ** -40 * lost
                off = (out[t].view(self.heads, self.d).double() - want).abs()
                assert bool((off <= bound).all()), (b, j, float((off / bound).max()))
                worst = max(worst, float((off / bound).max()))
        idle = [t for t in range(self.q.shape[0]) if t not in live]
        assert bool((out[idle] == 0).all())
        print(f"  worst {worst:.3f} of the bound", flush=True)
        return out


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("kind", ["tree", "chain", "any"])
def test_lengths_at_the_ends_of_tiles_and_pages(d, page, kind):
    held = [0, 0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 191, 250, 255, 257, 511, 513, 1000]
    counts = [1, 64, 1, 1, 2, 5, 64, 31, 1, 64, 3, 2, 63, 17, 9, 1, 33, 16, 15, 64]
    Case(8, 2, d, page, held, counts, kind=kind, refused=(4, 13), pad=3).check()


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (3, 1), (5, 1), (8, 8), (6, 2), (14, 2), (16, 1), (17, 1), (40, 2), (99, 3), (64, 8)])
@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 3, 1], [9, 4, 8], [16, 1, 7], [64, 30, 2]])
@pytest.mark.parametrize("d", [64, 128])
def test_groups_of_heads_and_sizes_of_trees(heads, kv, counts, d):
    """From a row to 2112 for a KV head of a request."""
    Case(heads, kv, d, 32, [40, 700, 0], counts, seed=kv).check()


@pytest.mark.parametrize("heads,kv,d,page,held,counts", [
    (32, 8, 128, 16, [385], [8]), (32, 8, 128, 16, [5000], [1]), (32, 8, 128, 16, [5000], [16]), (64, 8, 128, 256, [20000, 3], [64, 64]), (8, 8, 64, 32, [33000], [5]),
    (4, 1, 128, 128, [1, 70000, 700], [3, 2, 40]), (16, 4, 128, 16, [3000 + 37 * i for i in range(12)], [1 + i for i in range(12)]),
    (4, 2, 64, 16, [(7 * i) % 300 for i in range(700)], [i % 4 for i in range(700)]), (2, 1, 128, 64, [20 + i % 9 for i in range(1500)] + [9000], [1 + i % 2 for i in range(1501)])])
def test_long_and_uneven(heads, kv, d, page, held, counts):
    Case(heads, kv, d, page, held, counts).check()


def test_a_table_with_room_for_more_and_room_for_more_nodes():
    Case(8, 2, 128, 16, [700, 5, 1300], [9, 1, 20], max_pages=4096, nodes=64).check()


def test_more_nodes_than_are_allowed():
    Case(8, 2, 128, 16, [70, 5], [9, 8], nodes=8).check()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("counts", [[3, 8], [40, 64]])
def test_masks_that_leave_nothing(d, counts):
    """A request that held nothing and nodes that name none: zeros; on a request that held something the mask leaves that."""
    c = Case(4, 2, d, 16, [0, 20], counts)
    c.masks[0], c.masks[2], c.masks[counts[0] + 1] = 0, 0, 0
    out = c.check()
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all()) and bool((out[counts[0] + 1] != 0).any())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,counts", [(2, [4, 9]), (16, [64, 40])])
@pytest.mark.parametrize("value", [NAN, float("inf"), float("-inf"), -65504.0])
def test_what_is_masked_has_no_influence(d, heads, counts, value):
    """Keys, values, or both, of nodes that others do not see; of the places behind the last node; of pages that nobody holds."""
    c = Case(heads, 2, d, 16, [37, 0], counts, filler=value)
    last = counts[0] - 1                          # seen by itself alone
    for j in range(counts[0]):
        mask = c.masks[j] & (1 << last) - 1 if j < last else 1 << last
        c.masks[j] = mask - (1 << 64) if mask >> 63 else mask
    want = c.run()
    p = 37 + last
    for pages in ((c.kpages,), (c.vpages,), (c.kpages, c.vpages)):
        saved = [t.clone() for t in pages]
        for t in pages:
            t[c.rows[0][p // 16], :, p % 16] = value
        out = c.run()
        others = [t for t in range(c.q.shape[0]) if t != last]
        assert torch.equal(out[others].view(torch.int16), want[others].view(torch.int16))
        for t, old in zip(pages, saved):
            t.copy_(old)
    c.check()


def test_pages_that_do_not_exist_are_left_out():
    for number in (-1, 2 ** 31 - 1, None):
        c = Case(8, 2, 128, 16, [200, 40, 16], [9, 3, 2])
        for b, p in ((0, 3), (0, 12), (1, 0), (2, 0)):
            c.table[b][p] = c.kpages.shape[0] if number is None else number
        c.check(bad=[(b, p * 16 + i) for b, p in ((0, 3), (1, 0), (2, 0)) for i in range(16)] + [(0, 192 + i) for i in range(16) if 192 + i < 209])


def test_a_request_of_no_pages_at_all():
    c = Case(4, 2, 64, 16, [20], [3])
    c.table = [[-1] * 2]
    assert bool((c.run() == 0).all())


@pytest.mark.parametrize("where", ["q", "key", "value"])
@pytest.mark.parametrize("held,counts", [([300, 40], [6, 3]), ([3000, 40], [64, 3])])
def test_infinities_and_nan_that_are_seen(where, held, counts):
    """They reach the rows that see them, as in 64 bits, and no others."""
    c = Case(4, 2, 128, 16, held, counts)
    want = c.run()
    hit = torch.zeros_like(want, dtype=torch.bool).view(-1, 4, 128)
    if where == "q":
        c.q[1, 130] = NAN
        hit[1, 1] = True
        out = c.run().view(-1, 4, 128)
        assert bool(torch.isnan(out[hit]).all())
    elif where == "key":
        c.kpages[c.rows[0][2], 0, 5, 9] = NAN     # heads 0 and 1 of the first request
        hit[:counts[0], :2] = True
        out = c.run().view(-1, 4, 128)
        assert bool(torch.isnan(out[hit]).all())
    else:
        c.vpages[c.rows[0][2], 1, 5, 9] = float("inf")
        hit[:counts[0], 2:, 9] = True
        out = c.run().view(-1, 4, 128)
        assert bool((out[hit] == float("inf")).all())
    assert torch.equal(out[~hit], want.view(-1, 4, 128)[~hit]) or where != "q" and bool(((out[~hit] - want.view(-1, 4, 128)[~hit]).abs() <= 2.0 ** -9).all())


def test_keys_of_minus_infinity_weigh_nothing():
    c = Case(2, 1, 128, 16, [100], [4])
    c.q[:, :128], c.q[:, 128:] = c.q[:, :128].abs(), c.q[:, 128:].abs()
    saved = c.kpages.clone()
    c.kpages[c.rows[0][1], 0, 3] = float("-inf")
    out = c.run()
    c.kpages.copy_(saved)
    c.check(out, bad=[(0, 19)])


def test_weights_far_below_the_largest():
    """One score 20 above thousands of others, whose values are large: together they count."""
    c = Case(1, 1, 128, 16, [8000], [2])
    c.q.zero_()
    c.q[:, 0] = 16.0
    for p in range(8002):
        c.kpages[c.rows[0][p // 16], 0, p % 16, 0] = 0.0
    c.kpages[c.rows[0][0], 0, 0, 0] = 14.0        # a score of 19.8
    c.vpages[c.rows[0][0], 0, 0] = 0.0
    for p in range(1, 8000):
        c.vpages[c.rows[0][p // 16], 0, p % 16] = 60000.0
    out = c.check()
    assert float(out[0, 0]) > 1.0


def test_queries_with_rows_of_their_own_and_an_output_of_the_caller():
    c = Case(8, 2, 128, 16, [90, 5], [7, 2])
    want = c.run()
    wide = torch.zeros(9, 8 * 128 + 37, dtype=torch.float16, device="cuda")
    wide[:, 5:5 + 1024] = c.q
    c.q = wide[:, 5:5 + 1024]
    out = torch.full((9, 1024), NAN, dtype=torch.float16, device="cuda")
    assert c.run(out=out) is out and torch.equal(out.view(torch.int16), want.view(torch.int16))


def test_pages_beyond_32_bits():
    """A pool of more than 4 GiB, its last pages in use."""
    c = Case(4, 2, 128, 1024, [3000], [5], spare=8200, filler=0.0)
    assert c.kpages.numel() > 2 ** 31
    pool = c.kpages.shape[0]
    for i, row in enumerate(c.rows[0]):
        to = pool - 1 - i
        if to not in c.rows[0]:
            for t in (c.kpages, c.vpages):
                t[to].copy_(t[row])
            c.rows[0][i] = to
    c.table = [c.rows[0]]
    c.check()
    del c, t
    torch.cuda.empty_cache()


def test_the_same_bits_again():
    c = Case(16, 4, 128, 16, [900, 7000, 33], [9, 12, 64])
    want = c.run()
    for _ in range(5):
        assert torch.equal(c.run().view(torch.int16), want.view(torch.int16))


def test_no_rows():
    c = Case(4, 2, 64, 16, [20, 30], [0, 0], nodes=4)
    assert c.run().shape == (0, 256)
    c = Case(4, 2, 64, 16, [20], [0], nodes=4, pad=5)
    assert bool((c.run() == 0).all())


@pytest.mark.parametrize("kv,counts", [(8, 4), (16, 8), (16, 16), (16, 32)])
@pytest.mark.parametrize("held", [
    [400] * 10, [100, 7000] + [3] * 30, [900 - 60 * i for i in range(14)], [300] * 31 + [301], [700 * (i % 3) for i in range(60)], [1100] + [0] * 63, [40] * 65, [25 * (i % 40) for i in range(90)],
    [(37 * i) % 1500 for i in range(33)], [5] * 300 + [2500]])
def test_how_requests_are_dealt(kv, counts, held):
    """Few and many requests to a workgroup, alike and not: whole ones, own parts, equal shares."""
    Case(2 * kv, kv, 64, 16, held, [1 + (counts + i) % counts if i % 7 else 0 for i in range(len(held))], nodes=2 * counts if counts < 32 else 64, kind="chain").check()
