"""Requests that were granted more nodes than they have positions, which no plan leaves, have none: no positions and masks, zeros, nothing accepted.  The others' results are what they are without them."""
import random

import pytest
import torch

import tree_oracle as oracle
from paged_oracle import pages_of
from test_gpu_tree_accept import Case, on
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def numbers(B, seed):
    """(lengths, granted, those that are short): every third request has fewer positions than nodes."""
    rng = random.Random(seed)
    granted = [rng.choice((1, 2, 5, 9, 33, 64)) for _ in range(B)]
    short = range(0, B, 3)
    lengths = [rng.randrange(n) if b in short else n + rng.randrange(50) for b, n in enumerate(granted)]
    return lengths, granted, short


@pytest.mark.parametrize("B", [1, 5, 200])
def test_plan_and_attention(B):
    lengths, granted, short = numbers(B, B)
    starts = [sum(granted[:b]) for b in range(B + 1)]
    parents = [j - 1 for n in granted for j in range(n)]
    got = IU.tree_plan_hip(on(parents), on(lengths), on(granted), on(starts))
    positions, masks = oracle.plan(parents, lengths, [0 if b in short else n for b, n in enumerate(granted)], starts)
    held = [lengths[b] - n for b, n in enumerate(granted)]
    want = [-1 if b in short else held[b] + j for b, n in enumerate(granted) for j in range(n)]
    assert got.positions.tolist() == want
    assert got.masks.tolist() == masks
    wide = max(1, pages_of(max(lengths), 16))                             # (a table has a column)
    pool = B * wide
    table = torch.arange(pool, dtype=torch.int32, device="cuda").view(B, wide)
    k, v = torch.randn(2, pool, 1, 16, 64, device="cuda").half()
    q = torch.randn(starts[-1], 128, device="cuda").half()
    all_masks = torch.full((starts[-1],), -1, device="cuda")
    out = IU.attention_tree_hip(q, k, v, table, on(lengths), on(granted), on(starts), all_masks)
    for b, n in enumerate(granted):
        assert bool((out[starts[b]:starts[b + 1]] != 0).any()) == (b not in short)


@pytest.mark.parametrize("B", [1, 5, 64, 65, 300])
@pytest.mark.parametrize("inplace", [False, True])
def test_acceptance(B, inplace):
    _, granted, short = numbers(B, B)
    rng = random.Random(B)
    c = Case([rng.randrange(40) for _ in range(B)], granted, layers=2, kv=2, d=16, seed=B, agree=0.9)
    before = [rng.randrange(n) if b in short else c.lengths[b] for b, n in enumerate(granted)]
    c.table = [row[:pages_of(before[b], 16)] + [-5] * (len(row) - pages_of(before[b], 16)) for b, row in enumerate(c.table)]
    k, v = c.pages.clone()
    lengths, state, ring = on(before), on(c.state), on(c.ring)
    got = IU.tree_accept_hip(on(c.tokens, torch.int64), on(c.parents), on(c.targets, torch.int64), on(c.slots, torch.int64), lengths, on(granted), on(c.starts), on(c.table), ring, state, k, v,
                             64, inplace=inplace)
    # the oracle counts a request without nodes as one that keeps its positions: here they go back, all of them being new tokens'
    want = list(oracle.accept(c.tokens, c.parents, c.targets, c.lengths, [0 if b in short else n for b, n in enumerate(granted)], c.starts, c.table, c.ring, c.state, 16, 64))
    for b in range(B):
        if b in short:
            assert int(got.accepted[b]) == 0 and int(got.lengths[b]) == 0 and int(got.token[b]) == -1 and set(got.path[b].tolist()) == {-1}
        else:
            assert (int(got.lengths[b]), int(got.accepted[b]), got.path[b].tolist(), int(got.token[b])) == (want[0][b], want[2][b], want[3][b], want[4][b])
    (head, count), pool = c.state, len(c.ring)
    want_ring = list(c.ring)
    for b in range(B):
        for p in c.table[b][pages_of(got.lengths[b].item(), 16):pages_of(before[b], 16)]:
            want_ring[(head + count) % pool] = p
            count += 1
    assert ring.tolist() == want_ring and got.state.tolist() == [head, count]
    # the keys and values of all positions that somebody holds
    for t, old in ((k, c.pages[0]), (v, c.pages[1])):
        moved = oracle.moved(old, c.slots, c.starts, [[] if b in short else way for b, way in enumerate(want[3])], 16)
        for b in range(B):
            for at in range(0, int(got.lengths[b]), 16):
                m = min(16, int(got.lengths[b]) - at)
                page = c.table[b][at // 16]
                assert torch.equal(t[:, page, :, :m], moved[:, page, :, :m])
