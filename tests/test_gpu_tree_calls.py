"""The operators for drafted trees, forked rows and settings on logits called in other ways than one after another: captured and replayed, two graphs at once, on other
streams, by several threads, with tensors that take the Python path, again and again, in a captured step of a decoder."""
import threading

import pytest
import torch

from bitstack_amd.utils import inference_utils as IU
from bitstack_amd.utils.llama_decode import PROJ, LlamaShape, PagedCache, SyntheticLlamaDecoder

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Trees:
    """Requests with held positions and trees that change from call to call."""

    def __init__(self, B, nodes, longest, seed, page=16):
        self.g, self.B, self.nodes, self.longest, self.page = gen(seed), B, nodes, longest, page
        i32 = dict(dtype=torch.int32, device="cuda")
        self.T = B * nodes
        self.lengths, self.granted, self.starts = torch.zeros(B, **i32), torch.zeros(B, **i32), torch.zeros(B + 1, **i32)
        self.parents = torch.zeros(self.T, **i32)
        self.max_pages = -(-(longest + nodes) // page)
        self.table = torch.randperm(B * self.max_pages, device="cuda", generator=self.g).int().view(B, -1)
        self.slots = torch.zeros(self.T, dtype=torch.int64, device="cuda")

    def change(self):
        counts = torch.randint(1, self.nodes + 1, (self.B,), dtype=torch.int32, device="cuda", generator=self.g)
        self.starts[1:].copy_(counts.cumsum(0))
        self.granted.copy_(counts * (torch.rand(self.B, device="cuda", generator=self.g) < 0.8))
        self.lengths.copy_(torch.randint(0, self.longest + 1, (self.B,), dtype=torch.int32, device="cuda", generator=self.g) + self.granted)
        row = torch.searchsorted(self.starts[1:].contiguous(), torch.arange(self.T, device="cuda"), right=True).clamp(max=self.B - 1)
        node = torch.arange(self.T, device="cuda") - self.starts[row]
        self.parents.copy_(node - 1 - (2 * torch.rand(self.T, device="cuda", generator=self.g)).int())
        at = (self.lengths - self.granted)[row].long() + node
        self.slots.copy_(torch.where(node < self.granted[row], self.table[row].gather(1, at.clamp(0, self.max_pages * self.page - 1)[:, None] // self.page)[:, 0].long() * self.page + at % self.page, -1))

    def changed(self):
        return ()


class Plan(Trees):
    def __init__(self, B, nodes):
        super().__init__(B, nodes, 500, B)
        self.change()

    def run(self):
        return tuple(IU.tree_plan_hip(self.parents, self.lengths, self.granted, self.starts))


class Attend(Trees):
    def __init__(self, B, nodes, longest, heads=8, kv=2, d=128):
        super().__init__(B, nodes, longest, B + nodes)
        self.q = torch.randn(self.T, heads * d, dtype=torch.float16, device="cuda", generator=self.g)
        self.kp, self.vp = torch.randn(2, self.table.numel(), kv, self.page, d, dtype=torch.float16, device="cuda", generator=self.g)
        self.masks = torch.zeros(self.T, dtype=torch.int64, device="cuda")
        self.change()

    def change(self):
        super().change()
        self.q.normal_(generator=self.g)
        self.masks.copy_(IU.tree_plan_hip(self.parents, self.lengths, self.granted, self.starts).masks)

    def run(self):
        return IU.attention_tree_hip(self.q, self.kp, self.vp, self.table, self.lengths, self.granted, self.starts, self.masks, self.nodes),


class Accept(Trees):
    def __init__(self, B, nodes, layers=2, kv=2, d=64):
        super().__init__(B, nodes, 60, B + nodes)
        pool = self.table.numel()
        self.ring, self.state = torch.zeros(pool, dtype=torch.int32, device="cuda"), torch.tensor([pool - 2, 0], dtype=torch.int32, device="cuda")
        self.kp, self.vp = torch.zeros(2, layers, pool, kv, self.page, d, dtype=torch.float16, device="cuda")
        self.tokens, self.targets = torch.zeros(2, self.T, dtype=torch.int64, device="cuda")
        self.change()

    def change(self):
        super().change()
        self.kp.normal_(generator=self.g)
        self.vp.normal_(generator=self.g)
        self.tokens.random_(0, 2, generator=self.g)
        self.targets.random_(0, 2, generator=self.g)
        self.state[1] = 0

    def run(self):
        return tuple(IU.tree_accept_hip(self.tokens, self.parents, self.targets, self.slots, self.lengths, self.granted, self.starts, self.table, self.ring, self.state, self.kp, self.vp,
                                        self.nodes))

    def changed(self):
        return self.ring, self.kp, self.vp


class Fork:
    """Rows that become copies of each other, again and again, in place."""

    def __init__(self, B, max_pages, layers=2, kv=1, d=64, page=16):
        self.g, self.B = gen(B), B
        pool = B * max_pages + 3
        i32 = dict(dtype=torch.int32, device="cuda")
        self.lengths = torch.randint(0, max_pages * page + 1, (B,), generator=self.g, **i32)
        held = (self.lengths + page - 1) // page
        self.table = torch.arange(B * max_pages, **i32).view(B, max_pages)
        free = torch.cat([self.table[torch.arange(max_pages, device="cuda") >= held[:, None]], torch.arange(B * max_pages, pool, **i32)])
        self.ring, self.state = torch.zeros(pool, **i32), torch.tensor([0, free.numel()], **i32)
        self.ring[:free.numel()] = free
        self.shares, self.source = torch.zeros(pool, **i32), torch.zeros(B, **i32)
        self.kp, self.vp = torch.randn(2, layers, pool, kv, page, d, dtype=torch.float16, device="cuda", generator=self.g)
        self.change()

    def change(self):
        self.source.random_(0, self.B, generator=self.g)
        self.source[0] = 0
        self.source[self.B // 2] = -1

    def run(self):
        return IU.page_fork_hip(self.source, self.lengths, self.table, self.ring, self.state, self.shares, self.kp, self.vp, inplace=True).granted,

    def changed(self):
        return self.lengths, self.table, self.ring, self.state, self.shares, self.kp, self.vp


class Adjust:
    def __init__(self, R, V, most):
        self.g, self.R, self.V = gen(V), R, V
        self.x = torch.zeros(R, V, dtype=torch.float16, device="cuda")
        i32 = dict(dtype=torch.int32, device="cuda")
        self.s = {"history": torch.zeros(R, most, **i32), "history_lengths": torch.zeros(R, **i32), "prompt_lengths": torch.zeros(R, **i32), "bias_tokens": torch.zeros(R, 9, **i32),
                  "allowed": torch.zeros(2, -(-V // 32), **i32), "allowed_rows": torch.zeros(R, **i32)}
        self.s.update({name: torch.rand(R, device="cuda", generator=self.g) + 0.5 for name in ("repetition", "frequency", "presence")}, bias=torch.randn(R, 9, device="cuda", generator=self.g))
        self.change()

    def change(self):
        self.x.normal_(generator=self.g)
        for name, hi in (("history", self.V), ("history_lengths", self.s["history"].shape[1] + 1), ("prompt_lengths", 50), ("bias_tokens", self.V), ("allowed", 2 ** 31 - 1), ("allowed_rows", 2)):
            self.s[name].random_(0, hi, generator=self.g)

    def run(self):
        return IU.logits_adjust_hip(self.x, out=torch.empty_like(self.x), **self.s),

    def changed(self):
        return ()


KINDS = {"plan": lambda: Plan(20, 64), "attention, whole requests": lambda: Attend(5, 6, 200), "attention, 16 rows": lambda: Attend(3, 4, 3000), "attention, 32 rows": lambda: Attend(3, 8, 3000),
         "attention, 64 rows": lambda: Attend(3, 16, 3000), "attention, 128 rows": lambda: Attend(3, 32, 3000), "attention, 256 rows": lambda: Attend(3, 64, 2000),
         "attention, many requests": lambda: Attend(90, 3, 400), "accept": lambda: Accept(5, 20), "accept in two launches": lambda: Accept(70, 6), "fork": lambda: Fork(6, 5),
         "fork, many entries": lambda: Fork(40, 100, layers=1, d=8), "adjust": lambda: Adjust(3, 20000, 300)}


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b, strict=True))


@pytest.mark.parametrize("kind", KINDS)
def test_captured_and_replayed(kind):
    """Six replays with other inputs, each against the eager call on a case beside it, with eager work of the same kind in between."""
    case, eager, other = KINDS[kind](), KINDS[kind](), KINDS[kind]()
    other.run()
    before = [t.clone() for t in case.changed()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = case.run()
    assert same(before, case.changed())                  # capturing runs nothing
    for i in range(6):
        graph.replay()
        want = eager.run()
        assert same(got, want), i
        assert same(case.changed(), eager.changed()), i
        for c in (case, eager, other):
            c.change()
        other.run()


@pytest.mark.parametrize("kind", KINDS)
def test_two_graphs_at_once(kind):
    """Two graphs that torch captured on the same stream, replayed on two others at once."""
    cases, graphs, results = [KINDS[kind]() for _ in range(2)], [], []
    eager = [KINDS[kind]() for _ in range(2)]
    eager[0].run(), cases[0].run()
    for c in (cases[1], eager[1]):
        for _ in range(3):
            c.change()
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(c.run())
    streams = [torch.cuda.Stream() for _ in cases]
    for i in range(10):
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, e, r in zip(cases, eager, results):
            assert same(r, e.run()), i
            assert same(c.changed(), e.changed()), i
            c.change()
            e.change()


@pytest.mark.parametrize("kind", KINDS)
def test_on_other_streams(kind):
    """Threads with a stream each, and several with one; the results are those of the calls one after another."""
    rounds, workers = 10, 4
    cases, want = [KINDS[kind]() for _ in range(workers)], [KINDS[kind]() for _ in range(workers)]
    for i in range(workers):
        for _ in range(i):
            cases[i].change()
            want[i].change()
    results = [[] for _ in cases]
    torch.cuda.synchronize()
    shared = torch.cuda.Stream()
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), shared, shared]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(rounds):
                results[i].append([t.clone() for t in cases[i].run()])
                cases[i].change()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(workers)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(workers):
        for r in range(rounds):
            assert same(results[i][r], want[i].run()), (i, r)
            want[i].change()
        assert same(cases[i].changed(), want[i].changed())


class Other(torch.Tensor):
    """A tensor that is none of torch's own types."""


@pytest.mark.parametrize("kind", KINDS)
def test_python_path(kind, monkeypatch):
    """Tensors of a class of their own take the Python layer's path: the same results, captured too."""
    case, want = KINDS[kind](), KINDS[kind]()
    calls, require = [], IU._lib.require_gpu
    monkeypatch.setattr(IU._lib, "require_gpu", lambda *a: calls.append(1) or require(*a))
    name = {Plan: "parents", Attend: "kp", Accept: "tokens", Fork: "source", Adjust: "x"}[type(case)]
    setattr(case, name, getattr(case, name).as_subclass(Other))
    assert same(case.run(), want.run()) and same(case.changed(), want.changed())
    assert len(calls) == 1
    for c in (case, want):
        c.change()
    if type(case) is Attend:                              # (its change() calls tree_plan_hip)
        assert len(calls) == 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = case.run()
    for _ in range(3):
        graph.replay()
        assert same(got, want.run()) and same(case.changed(), want.changed())
        for c in (case, want):
            c.change()


@pytest.mark.parametrize("kind", [k for k in KINDS if "accept" not in k and "fork" not in k])
def test_again_and_again(kind):
    """The same call gives the same bits."""
    case = KINDS[kind]()
    first = [t.clone() for t in case.run()]
    for _ in range(20):
        assert same(case.run(), first)


SHAPE = LlamaShape(layers=2, hidden=512, intermediate=1024, heads=4, kv_heads=2, vocab=1000)
CONFIG = {f"layer.{L}.{p}": 2 + (L + j) % 2 for L in range(2) for j, p in enumerate(PROJ)}


@pytest.mark.parametrize("nodes", [5, 20])
def test_a_captured_step_with_drafts(nodes):
    """A whole step with trees (few tokens, and many), settings and draws in a graph, replayed with eager steps of another cache in between, against eager steps."""
    decs = [SyntheticLlamaDecoder(SHAPE, CONFIG, 512, "cuda", seed=5) for _ in range(2)]
    rows, g = 3, gen(1)
    caches = []
    for dec in decs:
        cache = PagedCache(dec, rows, pool_pages=100, forks=True)
        for row in range(rows):
            dec.prefill_paged(cache, row, torch.arange(10 + 7 * row, device="cuda") * 13 % 1000)
        cache.token.copy_(torch.tensor([1, 2, 3], device="cuda"))
        caches.append(cache)
    T = rows * nodes
    tokens = torch.zeros(T, dtype=torch.int64, device="cuda")
    parents = ((torch.arange(T, device="cuda") % nodes + 1) // 2 - 1).int()
    counts = torch.full((rows,), nodes, dtype=torch.int32, device="cuda")
    uniform = torch.zeros(T, device="cuda")
    adjust = dict(history=torch.randint(0, 1000, (rows, 50), dtype=torch.int32, device="cuda", generator=g), repetition=torch.full((rows,), 1.2, device="cuda"))
    temperature = torch.tensor([0.5, 1.0, 0.1], device="cuda")

    def step(i):
        plan, done, ids = decs[i].step_tree(caches[i], tokens, parents, counts, nodes=nodes, uniform=uniform, adjust=adjust, temperature=temperature)
        return done.path, done.token, ids, decs[i].logits

    def change():
        tokens.random_(0, 1000, generator=g)
        uniform.uniform_(generator=g)

    change()
    for i in range(2):                                    # (limits of LDS are raised, argument blocks made)
        step(i)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(0)
    for _ in range(5):
        change()
        graph.replay()
        assert same(got, step(1))
        assert same([getattr(caches[0], n) for n in ("lengths", "token", "free_state", "kpages")], [getattr(caches[1], n) for n in ("lengths", "token", "free_state", "kpages")])
