"""attention_paged_hip against attention in 64 bits, request by request.

The bound of an output o = sum_j w_j v_j: its rounding to fp16 (2^-11 |o|, or half of the smallest step), scores off by at most e (weights then by 2 e, and
the output by 2 e sum_j w_j |v_j|), the sums' own roundings in fp32 (chains of at most 2^9 steps: 2^-15) and what the second fp16 term of a weight cuts off
(2^-25 of the largest weight per position).  With tables that turn nothing the queries are exact, and e is the fp32 sum of d <= 128 products,
2^-17 sum |q k| / sqrt(d), and the scaling of the exponent, 2^-22 |s|; where the tables turn, also the rounding of the step's own key (2^-11 sum |q k| / sqrt(d); the
queries keep 2^-22)."""
import pytest
import torch

import paged_oracle as oracle
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, heads, kv, d, page, lengths, seed=0, turned=False, idle=(), spare=2, filler=float("nan"), max_pages=None):
        g = torch.Generator(device="cuda").manual_seed(seed + heads + d)
        self.heads, self.kv, self.d, self.page, self.idle = heads, kv, d, page, idle
        B = len(lengths)
        held = [oracle.pages_of(n, page) for n in lengths]
        self.pool = sum(held) + spare
        max_pages = max_pages or max(1, max(held))
        order = torch.randperm(self.pool, generator=torch.Generator().manual_seed(seed)).tolist()
        self.rows, at = [], 0
        for h in held:
            self.rows.append(order[at:at + h])
            at += h
        i32 = dict(dtype=torch.int32, device="cuda")
        self.table = torch.tensor([r + [-1] * (max_pages - len(r)) for r in self.rows], **i32)
        self.lengths = torch.tensor(lengths, **i32)
        self.slots = torch.tensor([-1 if n == 0 or b in idle else self.rows[b][(n - 1) // page] * page + (n - 1) % page for b, n in enumerate(lengths)], device="cuda")
        self.qkv = torch.randn(B, (heads + 2 * kv) * d, device="cuda", generator=g).half()
        self.qkv[:, :heads * d] *= 1.5
        # what nobody has written is no number
        self.kpages, self.vpages = torch.full((2, self.pool, kv, page, d), filler, device="cuda", dtype=torch.float16)
        for b, n in enumerate(lengths):
            for pages in (self.kpages, self.vpages):
                for p in range(oracle.pages_of(n - 1, page)):
                    m = min(page, n - 1 - p * page)
                    pages[self.rows[b][p], :, :m] = torch.randn(kv, m, d, device="cuda", generator=g).half()
        longest = max(max(lengths), 1)
        angles = torch.rand(longest, d // 2, device="cuda", generator=g) * 6.28 if turned else torch.zeros(longest, d // 2, device="cuda")
        self.cos, self.sin, self.turned = angles.cos().half(), angles.sin().half(), turned

    def args(self):
        return self.qkv, self.kpages, self.vpages, self.cos, self.sin, self.table, self.lengths, self.slots, self.heads, self.kv

    def run(self, **more):
        return IU.attention_paged_hip(*self.args(), **more)

    def live(self):
        return [b for b, s in enumerate(self.slots.tolist()) if s >= 0]

    def check(self, out, before):
        """out and the pages after a call, of which `before` holds copies from in front of it."""
        heads, kv, d, page = self.heads, self.kv, self.d, self.page
        written = torch.zeros(self.pool, page, dtype=torch.bool, device="cuda")
        worst = 0.0
        for b, n in enumerate(self.lengths.tolist()):
            got = out[b].view(heads, d)
            if b not in self.live():
                assert bool((got == 0).all()), b
                continue
            x = self.qkv[b].view(-1, d)
            q, own = oracle.rotate(x[:heads], self.cos[n - 1], self.sin[n - 1]), oracle.rotate(x[heads:heads + kv], self.cos[n - 1], self.sin[n - 1])
            p, o = self.rows[b][(n - 1) // page], (n - 1) % page
            written[p, o] = True
            assert bool(((self.kpages[p, :, o].double() - own).abs() <= 2.0 ** -11 * own.abs() + 2.0 ** -20).all())
            assert torch.equal(self.vpages[p, :, o], x[heads + kv:])
            keys, values = (torch.cat([t[r] for r in self.rows[b]], 1).transpose(0, 1)[:n - 1].double() for t in before)
            keys, values = torch.cat([keys, own[None]]), torch.cat([values, x[None, heads + kv:].double()])
            want, spread, size, lost = oracle.attend(q, keys, values, kv)
            e = (2.0 ** -16 + (2.0 ** -11 if self.turned else 0.0)) * size + 2.0 ** -20
            bound = 2.0 ** -11 * want.abs() + 2.0 ** -25 + (2 * e + 2.0 ** -14) * spread + lost
            off = (got.double() - want).abs()
            assert bool((off <= bound).all()), (b, n, float((off / bound).max()))
            worst = max(worst, float((off / bound).max()))
        for pages, old in ((self.kpages, before[0]), (self.vpages, before[1])):
            rest = ~written[:, None, :, None].expand_as(pages)
            assert torch.equal(pages[rest].view(torch.int16), old[rest].view(torch.int16))
        return worst


def check(*args, **more):
    print("paged attention", args, more, flush=True)
    c = Case(*args, **more)
    before = c.kpages.clone(), c.vpages.clone()
    out = c.run()
    worst = c.check(out, before)
    again = c.run()
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    print(f"  worst {worst:.3f} of the bound", flush=True)
    return c


EDGES = [1, 2, 0, 15, 16, 17, 18, 31, 33, 64, 127, 129, 130, 255, 257, 511, 513, 514]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("cut", [False, True])
def test_lengths_at_the_ends_of_tiles_and_pages(d, page, turned, cut):
    """Short tables are not cut, longer ones are, whatever the lengths."""
    check(8, 2, d, page, EDGES, turned=turned, idle=(5, 9), max_pages=1 + 1024 // page if cut else None)


@pytest.mark.parametrize("heads,kv", [(8, 8), (6, 2), (12, 1), (32, 4), (20, 1)])
@pytest.mark.parametrize("longest", [767, 768, 769, 1023, 1024, 1025])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_tables_around_the_longest_that_are_not_cut(heads, kv, longest, rows):
    check(heads, kv, 128, 16, [longest if b == 0 else (37 * b) % longest for b in range(rows)], seed=rows)


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (3, 1), (5, 1), (8, 8), (6, 2), (14, 2), (16, 1), (17, 1), (32, 1), (40, 2), (99, 3), (64, 8)])
@pytest.mark.parametrize("d", [64, 128])
def test_groups_of_heads(heads, kv, d):
    check(heads, kv, d, 32, [1, 40, 700, 0, 1111], seed=kv)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (8, 8), (14, 2), (17, 1), (40, 2), (64, 8)])
@pytest.mark.parametrize("rows", [1, 4, 20])
def test_groups_of_heads_in_short_tables(heads, kv, rows):
    check(heads, kv, 128, 16, [(500, 1, 40, 0, 333)[b % 5] + b // 5 for b in range(rows)], seed=rows)


# one long request, long and short ones together, many (more than one workgroup has threads), very many short ones
@pytest.mark.parametrize("heads,kv,d,page,lengths", [
    (32, 8, 128, 16, [385]), (32, 8, 128, 16, [5000]), (64, 8, 128, 256, [20000, 3]), (8, 8, 64, 32, [33000]), (4, 1, 128, 128, [1, 70000, 700]),
    (16, 4, 128, 16, [3000 + 37 * i for i in range(12)]), (4, 2, 64, 16, [(7 * i) % 300 for i in range(700)]), (2, 1, 128, 64, [20 + i % 9 for i in range(1500)] + [9000]),
    (20, 1, 128, 16, [1025, 2049, 513])])
def test_long_and_uneven(heads, kv, d, page, lengths):
    check(heads, kv, d, page, lengths)


def test_a_table_with_room_for_more():
    """Far more entries than any request holds: the split goes by the lengths."""
    check(8, 2, 128, 16, [700, 5, 1300], max_pages=4096)


def test_strided_rows_and_a_given_output():
    c = Case(8, 2, 128, 16, [100, 7, 0, 600], turned=True)
    wide = torch.randn(4, 12 * 128 + 24, device="cuda").half()
    wide[:, :12 * 128] = c.qkv
    plain = c.run()
    c.qkv = wide[:, 3:3 + 12 * 128].copy_(c.qkv.clone())
    out = torch.full((4, 8 * 128), 9.0, device="cuda", dtype=torch.float16)
    assert c.run(out=out) is out and torch.equal(out, plain)


def test_rows_that_are_idle():
    """No slot, a slot that does not exist, a length of 0, below, beyond the table's row, beyond the positions: zeros, and nothing is written."""
    c = Case(8, 2, 128, 16, [100, 100, 100, 100, 100, 1000, 100])
    before = c.kpages.clone(), c.vpages.clone()
    c.slots[1], c.slots[2] = c.pool * 16, 2 ** 45
    c.lengths[3], c.lengths[4] = 0, -3
    c.lengths[6] = 63 * 16 + 1
    c.slots[0] = -2 ** 40
    out = c.run()
    for b in (0, 1, 2, 3, 4, 6):
        assert bool((out[b] == 0).all()), b
    p = c.rows[5][999 // 16]
    for pages, old in ((c.kpages, before[0]), (c.vpages, before[1])):
        same = pages.view(torch.int16) == old.view(torch.int16)
        same[p, :, 999 % 16] = True
        assert bool(same.all())
    c.lengths[6], c.cos, c.sin = 999, c.cos[:500], c.sin[:500]
    out = c.run()
    assert bool((out[5:] == 0).all())


def test_entries_that_are_no_pages_are_left_out():
    c = Case(4, 2, 128, 16, [200, 700])
    for entry in (-1, c.pool, 2 ** 31 - 1, -2 ** 31):
        c.table[0, 3], c.table[1, 0], c.table[1, 40] = entry, entry, entry
        kpages, vpages = c.kpages.clone(), c.vpages.clone()
        out = c.run()
        for b, n in ((0, 200), (1, 700)):
            x = c.qkv[b].view(-1, 128)
            kept = [p for p in range(n - 1) if 0 <= int(c.table[b, p // 16]) < c.pool]
            at = torch.tensor(kept, device="cuda")
            ids = c.table[b][at // 16].long()
            keys = torch.cat([kpages[ids, :, at % 16], x[None, 4:6]])
            values = torch.cat([vpages[ids, :, at % 16], x[None, 6:]])
            want, spread, size, lost = oracle.attend(x[:4], keys, values, 2)
            bound = 2.0 ** -11 * want.abs() + 2.0 ** -25 + (2 * (2.0 ** -16 * size + 2.0 ** -20) + 2.0 ** -14) * spread + lost
            assert bool(((out[b].view(4, 128).double() - want).abs() <= bound).all())


def test_shared_pages():
    """Two requests with one prefix."""
    c = Case(4, 2, 128, 16, [64 + 9, 64 + 20])
    for pages in (c.kpages, c.vpages):
        for p in range(4):
            pages[c.rows[1][p]] = float("nan")
    c.table[1, :4] = c.table[0, :4]
    c.rows[1][:4] = c.rows[0][:4]
    before = c.kpages.clone(), c.vpages.clone()
    c.check(c.run(), before)


def test_infinite_values_and_large_scores():
    """A v of infinity gives infinity where its weight is not zero and leaves other heads and dimensions alone; scores of thousands leave one position."""
    c = Case(4, 2, 128, 16, [300, 40], filler=0.0)
    c.vpages[c.rows[0][2], 0, 5, 17] = float("inf")
    c.vpages[c.rows[0][9], 1, 3, 90] = float("-inf")
    out = c.run()
    flat = out[0].view(2, 2, 128)
    assert bool((flat[0, :, 17] == float("inf")).all()) and bool((flat[1, :, 90] == float("-inf")).all())
    flat[0, :, 17], flat[1, :, 90] = 0.0, 0.0
    assert bool(torch.isfinite(flat).all()) and bool(torch.isfinite(out[1]).all())
    c = Case(4, 2, 128, 16, [300, 40], filler=0.0)
    c.qkv[:, :4 * 128] *= 300.0
    before = c.kpages.clone(), c.vpages.clone()
    c.check(c.run(), before)


def test_pool_beyond_32_bits_of_values():
    """Pages behind 2^31 values of a pool."""
    kv, page, d = 1, 1024, 128
    pool = 2 ** 31 // (page * d) + 40
    c = Case(4, kv, d, page, [2500, 1025], spare=0)
    big = torch.zeros(2, pool, kv, page, d, device="cuda", dtype=torch.float16)
    shift = pool - c.pool
    big[0, shift:], big[1, shift:] = c.kpages, c.vpages
    small = c.run()
    c.kpages, c.vpages = big[0], big[1]
    c.table = torch.where(c.table >= 0, c.table + shift, c.table)
    c.slots += shift * page
    assert torch.equal(c.run(), small)
