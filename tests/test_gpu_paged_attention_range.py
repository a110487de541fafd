"""attention_paged_hip at the ends of the numbers: weights far below the largest, queries beyond fp16 after their rotation, infinite keys and values, and the
builds for large pools.

Bounds as in test_gpu_paged_attention.py, but for what the second fp16 term of a weight cuts off: the largest weight is held as 2^15, and half of the smallest
step of fp16, 2^-25, is then 2^-40 of it per position."""
import pytest
import torch

import paged_oracle as oracle
from test_gpu_paged_attention import Case

pytestmark = pytest.mark.gpu

GROUPS = [(1, 1), (2, 1), (4, 1), (8, 1), (12, 1), (20, 1), (6, 2)]


def rows_of(c, b):
    """(keys, values) of request b in 64 bits, the step's own among them; its queries."""
    n = int(c.lengths[b])
    x = c.qkv[b].view(-1, c.d)
    q, own = oracle.rotate(x[:c.heads], c.cos[n - 1], c.sin[n - 1]), oracle.rotate(x[c.heads:c.heads + c.kv], c.cos[n - 1], c.sin[n - 1])
    keys, values = (torch.cat([t[r] for r in c.rows[b]], 1).transpose(0, 1)[:n - 1].double() for t in (c.kpages, c.vpages))
    return torch.cat([keys, own[None]]), torch.cat([values, x[None, c.heads + c.kv:].double()]), q


def near(c, out, b, want, spread, size, lost):
    e = 2.0 ** -16 * size + 2.0 ** -20
    bound = 2.0 ** -11 * want.abs() + 2.0 ** -25 + (2 * e + 2.0 ** -14) * spread + lost * 2.0 ** -15      # (`lost` is 2^-25 per position)
    off = (out[b].view(c.heads, c.d).double() - want).abs()
    assert bool((off <= bound).all()), (b, float((off / bound).max()))


@pytest.mark.parametrize("heads,kv,d", [(8, 2, 128), (4, 4, 64), (16, 1, 128), (20, 1, 64), (1, 1, 128)])
@pytest.mark.parametrize("n", [600, 5000, 40000])
@pytest.mark.parametrize("ahead", [9.0, 14.0, 16.0, 18.0, 22.0])
@pytest.mark.parametrize("sinks", [1, 8])
def test_small_weights_are_not_lost(heads, kv, d, n, ahead, sinks):
    """One position far ahead whose v is 0 (or one in each of the first eight tiles), all others small and alike: the result is the small ones' alone."""
    print(f"sinks heads={heads} kv={kv} d={d} n={n} ahead={ahead} sinks={sinks}", flush=True)
    c = Case(heads, kv, d, 16, [n], filler=0.0)
    g = torch.Generator(device="cuda").manual_seed(n)
    c.qkv.zero_()
    c.qkv[:, :heads * d].view(1, heads, d)[:, :, 0] = 8.0
    c.kpages.zero_()
    c.vpages.copy_(0.5 + torch.rand(c.vpages.shape, device="cuda", generator=g))
    for t in range(sinks):
        c.kpages[c.rows[0][t], :, 0, 0] = ahead * d ** 0.5 / 8.0
        c.vpages[c.rows[0][t], :, 0] = 0.0
    keys, values, q = rows_of(c, 0)
    near(c, c.run(), 0, *oracle.attend(q, keys, values, kv))


@pytest.mark.parametrize("heads,kv", GROUPS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("longest", [500, 3000])
def test_queries_beyond_fp16(heads, kv, d, longest):
    """Two halves of 60000 rotated by an eighth of a turn are 0 and 84853: finite, as their scores are; and queries near the smallest fp16 numbers with large keys."""
    for scale, key in ((60000.0, 2e-4), (1e-5, 3e4)):
        c = Case(heads, kv, d, 16, [longest, 17, 1], filler=0.0)
        g = torch.Generator(device="cuda").manual_seed(longest + heads)
        c.cos.fill_(0.5 ** 0.5)
        c.sin.fill_(0.5 ** 0.5)
        q = torch.randn(3, heads, d, device="cuda", generator=g).clamp(-1, 1) * scale
        q[:, 0] = scale * (torch.rand(3, d, device="cuda", generator=g) < 0.5)
        c.qkv[:, :heads * d] = q.view(3, -1).half()
        c.qkv[:, heads * d:(heads + kv) * d] = 0.0                        # (its own key is not rounded)
        c.kpages.copy_(torch.randn(c.kpages.shape, device="cuda", generator=g).clamp(-2, 2) * key)
        assert scale < 1 or float(oracle.rotate(q[0], c.cos[0], c.sin[0]).abs().max()) > 65504
        out = c.run()
        for b in range(3):
            keys, values, q64 = rows_of(c, b)
            near(c, out, b, *oracle.attend(q64, keys, values, kv))


def without_weight(c, b, out):
    """Request b against the definition where keys hold infinities: a score of -inf is a weight of 0, one of +inf or NaN makes its head NaN."""
    keys, values, q = rows_of(c, b)
    rep, seen = c.heads // c.kv, set()
    for h in range(c.heads):
        hk, got = h // rep, out[b].view(c.heads, c.d)[h]
        s = (keys[:, hk] * q[h]).sum(1)
        if bool(torch.isnan(s).any()) or float(s.max()) == float("inf"):
            assert bool(torch.isnan(got).all()), (b, h)
            seen.add("nan")
            continue
        stays = s > -float("inf")
        want, spread, size, lost = oracle.attend(q[h:h + 1], keys[stays][:, hk:hk + 1], values[stays][:, hk:hk + 1], 1)
        bound = 2.0 ** -11 * want.abs() + 2.0 ** -25 + (2 * (2.0 ** -16 * size + 2.0 ** -20) + 2.0 ** -14) * spread + lost
        assert bool(((got.double() - want[0]).abs() <= bound[0]).all()), (b, h)
        seen.add("number")
    return seen


@pytest.mark.parametrize("heads,kv", GROUPS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("longest", [300, 2500])
def test_infinite_keys(heads, kv, d, longest):
    """Single keys, all keys of a tile, those of a wave's every tile, and all but the step's own; the sign of a query's element decides what an infinite one does to its head."""
    inf = float("inf")
    c = Case(heads, kv, d, 16, [longest, 40, 129, 40, longest, 40], filler=0.0, spare=1)
    c.qkv[:, :heads * d].view(6, heads, d)[:, :, 3].abs_().clamp_(min=0.25)        # one way for all heads ...
    c.qkv[:, :heads * d].view(6, heads, d)[4, ::2, 3] *= -1.0                     # ... but for these: their rows are NaN
    c.kpages[c.rows[0][0], :, 2, 3] = -inf
    c.kpages[c.rows[0][longest // 32], :, 7, 3] = -inf
    c.kpages[c.rows[1][0], :, :, 3] = -inf
    for p in c.rows[2]:
        c.kpages[p, :, :, 3] = -inf
    c.kpages[c.rows[3][1], :, 4, 3] = float("nan")
    c.kpages[c.rows[4][5], :, 9, 3] = -inf
    c.kpages[c.rows[5][2], :, 7, 3] = -inf                                        # (position 39 is the step's own: nobody reads what was there)
    out = c.run()
    assert without_weight(c, 0, out) == {"number"} and without_weight(c, 1, out) == {"number"} and without_weight(c, 2, out) == {"number"}
    assert without_weight(c, 3, out) == {"nan"} and without_weight(c, 5, out) == {"number"}
    assert without_weight(c, 4, out) == ({"number", "nan"} if heads > 1 else {"nan"})


@pytest.mark.parametrize("heads,kv", GROUPS)
@pytest.mark.parametrize("d", [64, 128])
def test_infinite_values_in_cut_requests(heads, kv, d):
    """A v of infinity in a request that is cut, and in one that is not beside it: infinity in its dimension for the heads that share it, all else as without it."""
    inf = float("inf")
    c = Case(heads, kv, d, 16, [4000, 700, 30], filler=0.0)
    plain = c.run()
    for b, p, at, dim, v in ((0, 3, 5, 17, inf), (0, 240, 2, 60, -inf), (1, 20, 0, 1, inf), (2, 0, 15, 33, -inf)):
        c.vpages[c.rows[b][p], 0, at, dim] = v
    out, rep = c.run().view(3, heads, d), heads // kv
    for b, dim, v in ((0, 17, inf), (0, 60, -inf), (1, 1, inf), (2, 33, -inf)):
        assert bool((out[b, :rep, dim] == v).all()), (b, dim)
        out[b, :rep, dim] = plain.view(3, heads, d)[b, :rep, dim]
    # the repeated sums are fp32 in another order, where a wave takes them: 2^-14 of the weights' sum of |v|, and a rounding to fp16
    assert bool(((out.double() - plain.view(3, heads, d).double()).abs() <= 2.0 ** -10 * plain.view(3, heads, d).double().abs() + 2.0 ** -12).all())


@pytest.mark.parametrize("heads,kv", GROUPS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths", [[300, 0, 1, 47], [3000, 20, 1025]])
def test_large_pools(heads, kv, d, lengths):
    """Pools from 256 MiB on are read past the last-level cache: the same bits as from a small pool, nothing read of what nobody has written."""
    c = Case(heads, kv, d, 64, lengths, turned=True)
    before = c.kpages.clone(), c.vpages.clone()
    small = c.run()
    c.check(small, before)
    pool = -(-2 ** 28 // (64 * kv * d * 4))
    order = torch.randperm(pool, device="cuda", generator=torch.Generator(device="cuda").manual_seed(d))[:c.pool]
    big = torch.full((2, pool, kv, 64, d), float("nan"), device="cuda", dtype=torch.float16)
    big[0, order], big[1, order] = before
    kpages = c.kpages
    c.kpages, c.vpages = big[0], big[1]
    c.table = torch.where(c.table >= 0, order[c.table.clamp(min=0).long()].int(), c.table)
    c.slots = torch.where(c.slots >= 0, order[c.slots.clamp(min=0) // 64] * 64 + c.slots % 64, c.slots)
    assert torch.equal(c.run().view(torch.int16), small.view(torch.int16))
    assert torch.equal(big[0, order].view(torch.int16), kpages.view(torch.int16))


def test_a_length_beyond_the_tables_row():
    """... is idle by that alone: the RoPE tables go further."""
    c = Case(8, 2, 128, 16, [100, 1000, 100])
    c.cos, c.sin = torch.ones(2000, 64, device="cuda", dtype=torch.float16), torch.zeros(2000, 64, device="cuda", dtype=torch.float16)
    before = c.kpages.clone(), c.vpages.clone()
    c.lengths[0] = 63 * 16 + 1
    out = c.run()
    assert bool((out[0] == 0).all()) and bool((out[1:] != 0).any(1).all())
    for pages, old in ((c.kpages, before[0]), (c.vpages, before[1])):
        p, o = c.rows[0][99 // 16], 99 % 16
        assert torch.equal(pages[p, :, o].view(torch.int16), old[p, :, o].view(torch.int16))
