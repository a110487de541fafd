"""step_paged() and prefill_paged() as a serving loop calls them: rows that are given back without a count of new tokens, vocabularies of any size, prompts in a
decoder with room for long ones."""
import pytest
import torch

from bitstack_amd.utils.llama_decode import PROJ, LlamaShape, PagedCache, SyntheticLlamaDecoder

CONFIG = {f"layer.{L}.{p}": 2 for L in range(2) for p in PROJ}


def decoder(vocab=1000, max_len=256):
    return SyntheticLlamaDecoder(LlamaShape(layers=2, hidden=512, intermediate=1024, heads=4, kv_heads=2, vocab=vocab), CONFIG, max_len, "cuda", seed=5)


def admit(dec, cache, *lengths):
    for row, n in enumerate(lengths):
        _, logits = dec.prefill_paged(cache, row, torch.randint(0, dec.s.vocab, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(row)))
        cache.token[row] = logits.argmax()


@pytest.mark.gpu
@pytest.mark.parametrize("max_len", [256, 250])
@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8])
def test_released_rows_take_no_new_token(max_len, dtype):
    """Without new_tokens: a row that gives its pages back is idle from then on, all others go on."""
    dec = decoder(max_len=max_len)
    cache = PagedCache(dec, 3, 40)
    admit(dec, cache, 20, 33, 16)
    tokens = cache.token.tolist()
    plan = dec.step_paged(cache, released=torch.tensor([0, 1, 0], device="cuda").to(dtype))
    assert plan.granted.tolist() == [1, 0, 1] and cache.lengths.tolist() == [21, 0, 17] and plan.row_slots.tolist()[1] == -1
    assert cache.token.tolist()[1] == tokens[1]
    assert cache.free_state.tolist()[1] == 40 - 2 - 2
    plan = dec.step_paged(cache, torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda"), released=torch.tensor([0, 0, 1], device="cuda").to(dtype))
    assert plan.granted.tolist() == [1, 1, 0] and cache.lengths.tolist() == [22, 1, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1003, 1002, 1004, 1000])
@pytest.mark.parametrize("rows", [1, 3, 9])
def test_greedy_with_any_vocabulary(vocab, rows):
    dec = decoder(vocab)
    cache = PagedCache(dec, rows, 40)
    admit(dec, cache, *(5 + 7 * b for b in range(rows)))
    for _ in range(3):
        dec.step_paged(cache)
        assert cache.token.tolist() == dec.logits.argmax(-1).tolist()


@pytest.mark.gpu
def test_a_prompt_takes_memory_by_its_length():
    """A short prompt of a decoder with room for 64 times as many positions allocates no more than one without."""
    peaks = []
    for max_len in (256, 16384):
        dec = decoder(max_len=max_len)
        cache = PagedCache(dec, 1, 16)
        admit(dec, cache, 100)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        admit(dec, cache, 100)
        peaks.append(torch.cuda.max_memory_allocated() - before)
    assert peaks[1] <= peaks[0] + (1 << 20), peaks


def test_settings_without_random_numbers_are_refused():
    """Greedy steps have no use for them: refused before anything is changed."""
    dec = SyntheticLlamaDecoder.__new__(SyntheticLlamaDecoder)
    for settings in (dict(temperature=1.0), dict(top_k=4), dict(top_p=None, min_p=0.1)):
        with pytest.raises(ValueError, match="uniform"):
            dec.step_paged(None, **settings)
