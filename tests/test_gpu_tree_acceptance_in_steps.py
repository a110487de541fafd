"""What step_tree accepts against a walk over the step's own logits, node by node: whole numbers, equal, so that a path that ends too early is found as well as one that goes too far."""
import random

import pytest
import torch

import tree_oracle as oracle
from test_gpu_tree_steps import One, decoder, drafts, i32, i64, prompt
from bitstack_amd.utils.llama_decode import PagedCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("right,wrong", [(3, 2), (0, 4), (6, 0), (9, 4)])
def test_paths_are_those_of_the_logits(page, right, wrong):
    rng, dec, rows = random.Random(page + right), decoder(), 3
    cache = PagedCache(dec, rows, pool_pages=4 + 700 // page, page_size=page)
    ones = []
    for row, n in enumerate((37, 16, 90)):
        p = prompt(n, row)
        _, logits = dec.prefill_paged(cache, row, p)
        cache.token[row] = logits.argmax()
        ones.append(One(p.tolist()))
    longest = 0
    for step in range(3):
        tokens, parents, counts = [], [], []
        for row in range(rows):
            t, p, _ = drafts(ones[row], int(cache.token[row]), rng, right, wrong) if row != step else ([], [], [])
            tokens, parents, counts = tokens + t, parents + p, counts + [len(t)]
        held, table, ring, state = cache.lengths.tolist(), cache.block_table.clone(), cache.free_pages.clone(), cache.free_state.clone()
        plan, done, ids = dec.step_tree(cache, i64(tokens), i32(parents), i32(counts))
        assert plan.granted.tolist() == counts and ids.tolist() == tokens
        targets = dec.logits.double().argmax(-1).tolist()
        lengths = [h + n for h, n in zip(held, counts)]
        want = oracle.accept(tokens, parents, targets, lengths, counts, plan.starts.tolist(), cache.block_table.tolist(), ring.tolist(), (int(state[0]), int(state[1])), page, 64)
        assert cache.lengths.tolist() == want[0] and done.accepted.tolist() == want[2] and done.path.tolist() == want[3]
        assert [int(cache.token[b]) for b in range(rows) if counts[b]] == [t for t, n in zip(want[4], counts) if n]
        longest = max(longest, max(want[2]))
        for row in range(rows):
            ones[row].text += [tokens[plan.starts[row] + j] for j in done.path[row].tolist() if j >= 0]
    # drafts that the model gives when it runs alone: as far as both runs agree, and they differ where the two largest logits are as good as equal alone
    assert longest > (right + 1) // 2
