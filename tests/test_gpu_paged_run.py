"""Requests of unequal lengths through a decoder: prompts come in, go on together, end and make room, over one pool of pages, against one decoder
per request with a cache of its own.

The tokens of the paged run are fed to the others too, so that the runs stay comparable: both are a few layers in fp16 with a dozen roundings each (2^-11 relative, of
either sign), by kernels that add in other orders for other batch sizes: sqrt(2 * 24) * 2^-11 = 3.4e-3 of the logits' norm, and 5e-3 is allowed."""
import pytest
import torch

from bitstack_amd.utils.llama_decode import PROJ, LlamaShape, PagedCache, SyntheticLlamaDecoder

pytestmark = pytest.mark.gpu

SHAPE = LlamaShape(layers=2, hidden=512, intermediate=1024, heads=4, kv_heads=2, vocab=1000)
CONFIG = {f"layer.{L}.{p}": 2 + (L + j) % 2 for L in range(2) for j, p in enumerate(PROJ)}


def decoder(batch=1, max_len=256):
    return SyntheticLlamaDecoder(SHAPE, CONFIG, max_len, "cuda", seed=5, batch=batch)


def prompt(n, seed):
    return torch.randint(0, SHAPE.vocab, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def near(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm()) <= 5e-3


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("sampled", [False, True])
def test_requests_come_and_go(page, sampled):
    dec, rows = decoder(), 4
    cache = PagedCache(dec, rows, pool_pages=3 + 400 // page, page_size=page)
    alone = {}                                             # row -> a decoder of its own
    live = torch.zeros(rows, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)

    def admit(row, n, seed):
        p = prompt(n, seed)
        plan, logits = dec.prefill_paged(cache, row, p)
        assert plan.granted.tolist() == [n if b == row else 0 for b in range(rows)]
        alone[row] = decoder()
        alone[row].prefill(p)
        assert near(logits[0], alone[row].logits[0])
        cache.token[row] = logits.argmax()
        live[row] = 1

    def step():
        released = (live == 0) & (cache.lengths > 0)
        for row, d in alone.items():
            d.token.copy_(cache.token[row:row + 1])
        if sampled:
            some = dict(temperature=torch.full((rows,), 0.8, device="cuda"), top_k=torch.full((rows,), 50, dtype=torch.int32, device="cuda"),
                        top_p=torch.full((rows,), 0.9, device="cuda"), min_p=torch.full((rows,), 0.02, device="cuda"))
            plan = dec.step_paged(cache, live, released=released, uniform=torch.rand(rows, device="cuda", generator=g), **some)
        else:
            plan = dec.step_paged(cache, live, released=released)
        assert plan.granted.tolist() == live.tolist()
        for row, d in alone.items():
            d.step_fused()
            assert near(dec.logits[row], d.logits[0]), row
            assert int(cache.lengths[row]) == int(d.pos)
            if not sampled:
                assert int(cache.token[row]) == int(dec.logits[row].argmax())
            assert 0 <= int(cache.token[row]) < SHAPE.vocab
        held = [-(-n // page) for n in cache.lengths.tolist()]
        pages = [p for b in range(rows) for p in cache.block_table[b, :held[b]].tolist()]
        assert len(set(pages)) == len(pages) and cache.free_state.tolist()[1] == cache.free_pages.numel() - len(pages)

    admit(0, 37, 1)
    admit(2, 100, 2)
    for _ in range(5):
        step()
    admit(3, 1, 3)
    for _ in range(20):
        step()
    live[2] = 0                                            # ends: its pages go back in the next step, its row stays idle
    del alone[2]
    for _ in range(3):
        step()
    assert int(cache.lengths[2]) == 0
    admit(2, 64, 4)
    admit(1, 17, 5)
    for _ in range(18):
        step()
    admit(0, 130, 6)                                       # a row taken up again at once
    for _ in range(3):
        step()


def test_as_decoders_in_lock_step():
    """All requests at one position: the decode step over pages gives what step_fused() gives over a cache [B, kv, max_len, d], whose kernels for the linears are the same."""
    B, n = 3, 45
    dec, paged = decoder(batch=B), decoder()
    cache = PagedCache(paged, B, 64)
    p = torch.stack([prompt(n, s) for s in range(B)])
    dec.prefill(p)
    for b in range(B):
        paged.prefill_paged(cache, b, p[b])
    cache.token.copy_(dec.token)
    for _ in range(10):
        dec.token.copy_(cache.token)
        paged.step_paged(cache)
        dec.step_fused()
        assert near(paged.logits, dec.logits)


def test_a_pool_that_runs_out():
    """The request that gets no page stays as it is and goes on when there is one again."""
    dec = decoder()
    cache = PagedCache(dec, 2, pool_pages=3)               # 48 positions
    for row, n in ((0, 16), (1, 31)):
        _, logits = dec.prefill_paged(cache, row, prompt(n, row))
        cache.token[row] = logits.argmax()
    before = cache.kpages.clone()
    plan = dec.step_paged(cache)                           # row 0 needs a page, row 1 has room for one more
    assert plan.granted.tolist() == [0, 1] and cache.lengths.tolist() == [16, 32] and plan.row_slots.tolist()[0] == -1
    pages = cache.block_table[0, :1].long()
    assert torch.equal(cache.kpages[:, pages], before[:, pages])
    token = int(cache.token[0])
    plan = dec.step_paged(cache, torch.tensor([1, 0], dtype=torch.int32, device="cuda"), released=torch.tensor([False, True], device="cuda"))
    assert plan.granted.tolist() == [0, 0] and int(cache.token[0]) == token
    plan = dec.step_paged(cache, torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
    assert plan.granted.tolist() == [1, 0] and cache.lengths.tolist() == [17, 0]
    alone = decoder()
    alone.prefill(prompt(16, 0))
    alone.token.fill_(token)
    alone.step_fused()
    assert near(dec.logits[0], alone.logits[0])
    _, _ = dec.prefill_paged(cache, 1, prompt(40, 9))
    assert cache.lengths.tolist() == [17, 0]               # three pages are needed, one is free


@pytest.mark.parametrize("max_len", [40, 48])
def test_up_to_the_last_position(max_len):
    """A request goes to the end of the RoPE tables, inside a page or at its end, and stays there; one that is given back there starts anew."""
    dec, alone = decoder(max_len=max_len), decoder(max_len=max_len)
    cache = PagedCache(dec, 2, 8)
    _, logits = dec.prefill_paged(cache, 1, prompt(max_len - 2, 3))
    alone.prefill(prompt(max_len - 2, 3))
    cache.token[1] = logits.argmax()
    live = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for i in range(4):
        token = int(cache.token[1])
        plan = dec.step_paged(cache, live)
        assert plan.granted.tolist() == [0, int(i < 2)] and int(cache.lengths[1]) == min(max_len, max_len - 1 + i)
        if i < 2:
            alone.token.fill_(token)
            alone.step_fused()
            assert near(dec.logits[1], alone.logits[0])
        else:
            assert int(cache.token[1]) == token
    plan = dec.step_paged(cache, live, released=live.bool())
    assert plan.granted.tolist() == [0, 1] and int(cache.lengths[1]) == 1


def test_a_captured_step():
    """step_paged() captured once and replayed: each replay is the eager step, across page ends and beside eager work."""
    eager, captured = decoder(), decoder()
    caches = [PagedCache(d, 3, 40) for d in (eager, captured)]
    for d, c in zip((eager, captured), caches):
        for row, n in enumerate((14, 50, 5)):
            _, logits = d.prefill_paged(c, row, prompt(n, row))
            c.token[row] = logits.argmax()
    g = torch.Generator(device="cuda").manual_seed(2)
    uniform = torch.rand(3, device="cuda", generator=g)
    settings = dict(temperature=torch.full((3,), 0.7, device="cuda"), top_p=torch.full((3,), 0.8, device="cuda"))
    live = torch.ones(3, dtype=torch.int32, device="cuda")
    for d, c in zip((eager, captured), caches):
        d.step_paged(c, live, uniform=uniform, **settings)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = caches[1]
        state = c.lengths, c.block_table, c.free_pages, c.free_state, c.token, c.kpages, c.vpages
        keep = [t.clone() for t in state]
        captured.step_paged(c, live, uniform=uniform, **settings)      # what it changed, the pages' new positions among it, is put back
        for t, k in zip(state, keep):
            t.copy_(k)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step_paged(caches[1], live, uniform=uniform, **settings)
    for i in range(40):
        uniform.copy_(torch.rand(3, device="cuda", generator=g))
        live[1] = 0 if i % 5 == 0 else 1
        graph.replay()
        eager.step_paged(caches[0], live, uniform=uniform, **settings)
        assert torch.equal(eager.logits, captured.logits)
        for a, b in zip((caches[0].lengths, caches[0].block_table, caches[0].free_pages, caches[0].free_state, caches[0].token, caches[0].kpages),
                        (caches[1].lengths, caches[1].block_table, caches[1].free_pages, caches[1].free_state, caches[1].token, caches[1].kpages)):
            assert torch.equal(a, b), i


def test_refusals():
    dec = decoder()
    cache = PagedCache(dec, 2, 8)
    for rows in (0, 49):
        with pytest.raises(ValueError):
            PagedCache(dec, rows, 8)
    with pytest.raises(ValueError):
        dec.prefill_paged(cache, 0, prompt(257, 0))
    with pytest.raises(ValueError):
        dec.prefill_paged(cache, 0, prompt(0, 0))
    for row in (-1, 2):
        with pytest.raises(ValueError, match="rows"):
            dec.prefill_paged(cache, row, prompt(3, 0))
    with pytest.raises(RuntimeError):
        dec.step_paged(PagedCache(dec, 2, 8, page_size=24))
    narrow = SyntheticLlamaDecoder(LlamaShape(layers=1, hidden=256, intermediate=512, heads=4, kv_heads=2, vocab=1000), CONFIG, 64, "cuda")
    with pytest.raises(ValueError, match="128"):
        narrow.prefill_paged(PagedCache(narrow, 1, 8), 0, prompt(3, 0))
