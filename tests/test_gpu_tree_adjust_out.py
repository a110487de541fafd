"""step_paged and step_tree with settings whose adjusted logits go to a tensor of the caller's: the tokens are drawn from those."""
import pytest
import torch

from test_gpu_tree_steps import SHAPE, decoder, i32, i64, prompt
from bitstack_amd.utils.llama_decode import PagedCache

pytestmark = pytest.mark.gpu


def cache_of(dec):
    cache = PagedCache(dec, 2, pool_pages=40)
    for row in range(2):
        _, logits = dec.prefill_paged(cache, row, prompt(20 + row, row))
        cache.token[row] = logits.argmax()
    return cache


def test_a_step_of_one_token():
    """A grammar that allows one token: greedy, it is the next one, and both results are those in place."""
    results = []
    for own in (False, True):
        dec = decoder()
        cache = cache_of(dec)
        allowed = torch.zeros(1, (SHAPE.vocab + 31) // 32, dtype=torch.int32, device="cuda")
        allowed[0, 7] = 1 << 5
        out = torch.zeros(2, SHAPE.vocab, dtype=torch.float16, device="cuda")
        dec.step_paged(cache, adjust=dict(allowed=allowed, allowed_rows=i32([0, -1]), **({"out": out} if own else {})))
        assert int(cache.token[0]) == 7 * 32 + 5
        assert not own or dec.logits is out
        results.append((dec.logits.clone(), cache.token.tolist()))
    assert torch.equal(results[0][0], results[1][0]) and results[0][1] == results[1][1]


def test_a_step_with_drafts():
    results = []
    for own in (False, True):
        dec = decoder()
        cache = cache_of(dec)
        history = i32([[3] * 8, [4] * 8])
        out = torch.zeros(6, SHAPE.vocab, dtype=torch.float16, device="cuda")
        bias = dict(bias_tokens=i32([[9], [8]]), bias=torch.full((2, 1), 2000.0, device="cuda"))
        _, done, ids = dec.step_tree(cache, i64([0, 9, 9, 0, 8, 7]), i32([-1, 0, 1] * 2), i32([3, 3]), adjust=dict(history=history, repetition=torch.full((2,), 1.2, device="cuda"), **bias,
                                                                                                                **({"out": out} if own else {})))
        assert done.accepted.tolist() == [3, 2] and cache.token.tolist() == [9, 8]
        results.append(dec.logits.clone())
    assert torch.equal(results[0], results[1])


@pytest.mark.parametrize("wide,first", [(SHAPE.vocab + 24, 0), (SHAPE.vocab + 24, 8), (SHAPE.vocab, 1), (SHAPE.vocab + 3, 2)])
def test_rows_of_a_wider_tensor(wide, first):
    """Greedy tokens from an output whose rows are apart, or do not start on 16 bytes."""
    results = []
    for own in (False, True):
        dec = decoder()
        cache = cache_of(dec)
        out = torch.zeros(2 * wide + first, dtype=torch.float16, device="cuda")[first:].view(2, wide)[:, :SHAPE.vocab]
        bias = dict(bias_tokens=i32([[9], [8]]), bias=torch.full((2, 1), 2000.0, device="cuda"))
        dec.step_paged(cache, adjust=dict(bias, **({"out": out} if own else {})))
        results.append((dec.logits.clone(), cache.token.tolist()))
    assert torch.equal(results[0][0], results[1][0]) and results[0][1] == results[1][1] == [9, 8]
