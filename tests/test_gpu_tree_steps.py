"""Drafted tokens, forked rows and settings on logits through a decoder, together, against steps of one token.

The runs differ by the order in which kernels add (other token counts take other kernels): sqrt(2 * 24) * 2^-11 = 3.4e-3 of the logits' norm for a few layers in fp16 with a dozen
roundings each, and 5e-3 is allowed; tokens are compared where the step of one token is sure of them by more than that."""
import random

import pytest
import torch

from bitstack_amd.utils.llama_decode import PROJ, LlamaShape, PagedCache, SyntheticLlamaDecoder

pytestmark = pytest.mark.gpu

SHAPE = LlamaShape(layers=2, hidden=512, intermediate=1024, heads=4, kv_heads=2, vocab=1000)
CONFIG = {f"layer.{L}.{p}": 2 + (L + j) % 2 for L in range(2) for j, p in enumerate(PROJ)}


def decoder(max_len=256, shape=SHAPE):
    return SyntheticLlamaDecoder(shape, CONFIG, max_len, "cuda", seed=5)


def prompt(n, seed, vocab=SHAPE.vocab):
    return torch.randint(0, vocab, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def near(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm()) <= 5e-3


def sure(logits):
    """Whether the largest is ahead by more than both runs' errors, twice 5e-3 of the norm."""
    top = logits.double().topk(2).values
    return float(top[0] - top[1]) > 1e-2 * float(logits.double().norm())


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def i64(v):
    return torch.tensor(v, dtype=torch.int64, device="cuda")


class One:
    """A request by itself, a token at a time: the text of any path of tokens behind its prompt has these logits."""

    def __init__(self, text, shape=SHAPE):
        self.dec, self.text, self.shape = decoder(shape=shape), list(text), shape

    def logits(self, path=()):
        self.dec.prefill(i64(self.text + list(path)))
        return self.dec.logits[0].clone()


def drafts(one, first, rng, right, wrong, vocab=SHAPE.vocab):
    """(tokens, parents): `right` tokens that the model gives, one behind the other, among others that it doesn't; and the path of the right ones."""
    tokens, parents, path, text = [first], [-1], [0], [first]
    for _ in range(right):
        best = int(one.logits(text).argmax())
        for _ in range(rng.randrange(wrong + 1)):
            tokens.append((best + 1 + rng.randrange(vocab - 1)) % vocab)
            parents.append(rng.randrange(len(tokens) - 1))
            if parents[-1] in path[:-1] and tokens[-1] == tokens[path[path.index(parents[-1]) + 1]]:
                tokens[-1] = (tokens[-1] + 1) % vocab
        tokens.append(best)
        parents.append(path[-1])
        path.append(len(tokens) - 1)
        text.append(best)
    return tokens, parents, path


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("right,wrong", [(3, 2), (0, 4), (6, 0), (9, 4)])
def test_drafts_are_accepted_as_far_as_they_are_right(page, right, wrong):
    """Three requests, one of them idle for a while; 1 to about 50 nodes each: both ways through the linear layers."""
    rng, dec, rows = random.Random(page + right), decoder(), 3
    cache = PagedCache(dec, rows, pool_pages=4 + 700 // page, page_size=page)
    ones = []
    for row, n in enumerate((37, 16, 90)):
        p = prompt(n, row)
        _, logits = dec.prefill_paged(cache, row, p)
        cache.token[row] = logits.argmax()
        ones.append(One(p.tolist()))
    for step in range(3):
        idle = step                               # this row has no tokens
        tokens, parents, counts, ways = [], [], [], []
        for row in range(rows):
            t, p, way = drafts(ones[row], int(cache.token[row]), rng, right, wrong) if row != idle else ([], [], [])
            tokens, parents, counts = tokens + t, parents + p, counts + [len(t)]
            ways.append((t, p, way))
        pad = 2
        before, firsts = cache.lengths.tolist(), cache.token.tolist()
        given = [7 if i in [sum(counts[:b]) for b in range(rows)] else t for i, t in enumerate(tokens)]        # (the first of a request is cache.token whatever stands there)
        plan, done, ids = dec.step_tree(cache, i64(given + [3] * pad), i32(parents + [0] * pad), i32(counts))
        assert ids.tolist()[:len(tokens)] == tokens
        for row in range(rows):
            t, p, way = ways[row]
            start = sum(counts[:row])
            if not t:
                assert int(done.accepted[row]) == 0 and int(cache.lengths[row]) == before[row] and int(cache.token[row]) == firsts[row]
                continue
            got = [j for j in done.path[row].tolist() if j >= 0]
            for j in range(len(t)):               # every node's logits are those of its path alone
                up, k = [], j
                while k >= 0:
                    up.append(t[k])
                    k = p[k]
                alone = ones[row].logits(up[::-1])
                assert near(dec.logits[start + j], alone), (row, j)
            assert len(got) == int(done.accepted[row]) and int(cache.lengths[row]) == before[row] + len(got)
            certain = [sure(ones[row].logits([t[k] for k in way[:i + 1]])) for i in range(len(way))]
            at = certain.index(False) if False in certain else len(way)
            assert got[:at + 1] == way[:at + 1] if at < len(way) else got == way
            new = [t[j] for j in got[1:]] + [int(cache.token[row])]
            assert all(int(dec.logits[start + j].argmax()) == token for j, token in zip(got, new))
            ones[row].text += [t[j] for j in got]
        held = [-(-n // page) for n in cache.lengths.tolist()]
        pages = [q for b in range(rows) for q in cache.block_table[b, :held[b]].tolist()]
        assert len(set(pages)) == len(pages) and cache.free_state.tolist()[1] == cache.free_pages.numel() - len(pages)
        # a step of one token goes on where the tree has left the cache
        live = i32([int(n > 0) for n in counts])
        firsts = cache.token.tolist()
        dec.step_paged(cache, live)
        for row in range(rows):
            if counts[row]:
                assert near(dec.logits[row], ones[row].logits([firsts[row]]))
                ones[row].text.append(firsts[row])


def test_requests_whose_pages_are_not_there():
    dec = decoder()
    cache = PagedCache(dec, 2, pool_pages=5)
    for row, n in enumerate((30, 30)):
        _, logits = dec.prefill_paged(cache, row, prompt(n, row))
        cache.token[row] = logits.argmax()
    first = cache.token.tolist()
    plan, done, _ = dec.step_tree(cache, i64([0] * 10), i32([-1, 0, 1, 2, 3] * 2), i32([5, 5]))
    assert plan.granted.tolist() == [5, 0] and done.accepted.tolist()[1] == 0 and cache.lengths.tolist()[1] == 30 and int(cache.token[1]) == first[1]
    assert int(cache.lengths[0]) == 30 + int(done.accepted[0]) and int(done.accepted[0]) >= 1


def test_drawn_tokens_and_settings():
    """A tree with temperature, penalties, biases and grammars: every node's logits are those that one row alone has with its own text, and what is drawn from them."""
    from bitstack_amd.utils import inference_utils as IU
    dec, rows, n = decoder(), 3, 6
    cache = PagedCache(dec, rows, pool_pages=60)
    texts = []
    for row, m in enumerate((20, 33, 47)):
        p = prompt(m, row)
        _, logits = dec.prefill_paged(cache, row, p)
        cache.token[row] = logits.argmax()
        texts.append(p.tolist() + [int(cache.token[row])])
    T = rows * n
    g = torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randint(0, SHAPE.vocab, (T,), device="cuda", generator=g)
    parents = i32([-1, 0, 0, 1, 3, 2] * rows)
    history = torch.zeros(rows, 64, dtype=torch.int32, device="cuda")
    for row, text in enumerate(texts):
        history[row, :len(text)] = i32(text)
    uniform = torch.rand(T, device="cuda", generator=g)
    adjust = dict(history=history, history_lengths=i32([len(t) for t in texts]), prompt_lengths=i32([20, 10, 47]), repetition=torch.tensor([1.3, 1.0, 0.8], device="cuda"),
                  frequency=torch.tensor([0.2, 0.5, 0.0], device="cuda"), presence=torch.tensor([0.0, 0.3, 0.7], device="cuda"), bias_tokens=i32([[5], [6], [7]]),
                  bias=torch.tensor([[2.0], [-3.0], [1.0]], device="cuda"), allowed=torch.randint(-2 ** 31, 2 ** 31, (4, 32), dtype=torch.int64, device="cuda", generator=g).int(),
                  allowed_rows=i32([(i * 5) % 5 - 1 for i in range(T)]))
    sampling = dict(temperature=torch.tensor([0.7, 1.0, 1.3], device="cuda"), top_k=i32([50, 0, 9]))
    plain = decoder()
    copy = PagedCache(plain, rows, pool_pages=60)
    for name in ("kpages", "vpages", "block_table", "lengths", "free_pages", "free_state", "token"):
        getattr(copy, name).copy_(getattr(cache, name))
    plain.step_tree(copy, tokens, parents, i32([n] * rows))
    raw = plain.logits.clone()
    _, done, ids = dec.step_tree(cache, tokens, parents, i32([n] * rows), uniform=uniform, adjust=adjust, **sampling)
    for t in range(T):
        row, up, k = t // n, [], t % n
        while k > 0:
            up.append(int(ids[row * n + k]))
            k = int(parents[row * n + k])
        text = i32(texts[row] + up[::-1])[None]
        alone = raw[t:t + 1].clone()
        one = {name: v[row:row + 1] for name, v in adjust.items() if name not in ("allowed", "history", "history_lengths", "allowed_rows")}
        IU.logits_adjust_hip(alone, history=text, history_lengths=i32([text.shape[1]]), allowed=adjust["allowed"], allowed_rows=adjust["allowed_rows"][t:t + 1], **one)
        assert torch.equal(alone[0], dec.logits[t]), t
    drawn = IU.sample_hip(dec.logits, uniform, temperature=sampling["temperature"].repeat_interleave(n), top_k=sampling["top_k"].repeat_interleave(n)).tolist()
    for row in range(rows):
        path = [j for j in done.path[row].tolist() if j >= 0]
        assert int(cache.token[row]) == drawn[row * n + path[-1]] and all(int(ids[row * n + b]) == drawn[row * n + a] for a, b in zip(path, path[1:]))


@pytest.mark.parametrize("page", [16, 64])
def test_forked_rows_go_on_by_themselves(page):
    """One prompt, four continuations that share its pages, an exchange of rows, ends; against each text alone."""
    dec, rows = decoder(), 4
    cache = PagedCache(dec, rows, pool_pages=6 + 500 // page, page_size=page, forks=True)
    p = prompt(75, 9)
    dec.prefill_paged(cache, 0, p)
    cache.token[0] = 11
    assert cache.fork(i32([0, 0, 0, 0])).granted.tolist() == [1] * 4 and cache.token.tolist() == [11] * 4
    texts = [p.tolist() for _ in range(rows)]
    cache.token.copy_(i64([11, 12, 13, 14]))

    def step(live, released=None):
        now = cache.token.tolist()
        dec.step_paged(cache, i32(live), released=released)
        for row in range(rows):
            if live[row]:
                texts[row].append(now[row])
                assert near(dec.logits[row], One(texts[row]).logits()), row
                assert int(cache.lengths[row]) == len(texts[row])

    for _ in range(3):
        step([1, 1, 1, 1])
    cache.fork(i32([2, 1, 0, -1]))
    texts = [texts[2], texts[1], texts[0], []]
    for _ in range(14):
        step([1, 1, 1, 0])
    step([1, 0, 1, 0], released=torch.tensor([False, True, False, False], device="cuda"))
    texts[1] = []
    plan, done, ids = dec.step_tree(cache, i64([0, 5, 6, 0, 7]), i32([-1, 0, 1, -1, 0]), i32([3, 0, 2, 0]))
    for row, at in ((0, 0), (2, 3)):
        texts[row] += [int(ids[at + j]) for j in done.path[row].tolist() if j >= 0]
    step([1, 0, 1, 0])
    cache.fork(i32([-1] * 4))
    assert cache.free_state.tolist()[1] == cache.free_pages.numel() and int(cache.shares.abs().sum()) == 0
    _, logits = dec.prefill_paged(cache, 3, p)             # the pages are there again
    assert near(logits[0], One(p.tolist()).logits())


def test_what_is_refused():
    dec = decoder(max_len=250)
    cache = PagedCache(dec, 2, pool_pages=40)
    with pytest.raises(ValueError, match="forks=True"):
        cache.fork(i32([0, 0]))
    with pytest.raises(ValueError, match="whole pages"):
        dec.step_tree(cache, i64([0]), i32([-1]), i32([1, 0]))
    dec = decoder()
    cache = PagedCache(dec, 2, pool_pages=40)
    with pytest.raises(ValueError, match="64 nodes"):
        dec.step_tree(cache, i64([0]), i32([-1]), i32([1, 0]), nodes=65)
    with pytest.raises(ValueError, match="a token at least"):
        dec.step_tree(cache, i64([]), i32([]), i32([0, 0]))
    with pytest.raises(ValueError, match="uniform"):
        dec.step_tree(cache, i64([0]), i32([-1]), i32([1, 0]), temperature=torch.ones(2, device="cuda"))


def test_a_request_ends_at_the_last_position():
    """A tree that does not fit is refused, one that does ends there."""
    dec = decoder(max_len=64)
    cache = PagedCache(dec, 1, pool_pages=8)
    _, logits = dec.prefill_paged(cache, 0, prompt(60, 1))
    cache.token[0] = logits.argmax()
    plan, done, _ = dec.step_tree(cache, i64([0] * 5), i32([-1, 0, 1, 2, 3]), i32([5]))
    assert plan.granted.tolist() == [0] and done.accepted.tolist() == [0] and cache.lengths.tolist() == [60]
    one = One(prompt(60, 1).tolist())
    t, p, way = drafts(one, int(cache.token[0]), random.Random(1), 3, 0)
    plan, done, _ = dec.step_tree(cache, i64(t), i32(p), i32([4]))
    assert plan.granted.tolist() == [4] and int(cache.lengths[0]) == 60 + int(done.accepted[0]) <= 64


@pytest.mark.parametrize("nodes", [4, 30])
def test_drafts_and_padding_that_are_no_tokens(nodes):
    """Rows of no request, and drafts, whose numbers are outside the vocabulary: the others' results are those with any token there, and such drafts are not accepted."""
    results = []
    for filler in (0, -1, 1 << 40):
        dec = decoder()
        cache = PagedCache(dec, 3, 60)
        for row in (0, 2):
            dec.prefill_paged(cache, row, prompt(20 + row, row))
        cache.token.copy_(i64([7, 8, 9]))
        T = 2 * nodes + 5
        tokens = torch.full((T,), filler, device="cuda")
        tokens[:2] = i64([7, 11])
        tokens[nodes] = 9
        parents = torch.arange(T, dtype=torch.int32, device="cuda") - 1
        parents[nodes:] -= nodes
        plan, done, ids = dec.step_tree(cache, tokens, parents, i32([nodes, 0, nodes]), nodes=nodes)
        assert plan.granted.tolist() == [nodes, 0, nodes]
        if filler:
            assert int(done.accepted[0]) <= 2 and int(done.accepted[2]) == 1
        results.append((dec.logits[:2].clone(), dec.logits[nodes].clone()))
    for got in results[1:]:
        assert torch.equal(got[0], results[0][0]) and torch.equal(got[1], results[0][1])
