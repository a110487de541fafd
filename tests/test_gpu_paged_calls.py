"""The operators for requests of unequal lengths called in other ways than one after another: captured and replayed, on other streams, at once,
with tensors that take the Python path, again and again."""
import threading

import pytest
import torch

from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Plan:
    """Lengths that grow, shrink (released) and cross page ends, from one call to the next."""

    def __init__(self, B, T, seed=0):
        self.g, self.B, self.T = gen(seed), B, T
        self.lengths = torch.randint(0, 200, (B,), dtype=torch.int32, device="cuda", generator=self.g)
        self.page, self.max_pages = 16, 64
        held = (self.lengths + 15) // 16
        ends = held.cumsum(0)
        self.table = torch.zeros(B, self.max_pages, dtype=torch.int32, device="cuda")
        for b in range(B):
            self.table[b, :held[b]] = torch.arange(int(ends[b] - held[b]), int(ends[b]), dtype=torch.int32, device="cuda")
        self.pool = int(ends[-1]) + 4 * B
        self.ring = torch.zeros(self.pool, dtype=torch.int32, device="cuda")
        self.ring[:4 * B] = torch.arange(int(ends[-1]), self.pool, dtype=torch.int32, device="cuda")
        self.state = torch.tensor([0, 4 * B], dtype=torch.int32, device="cuda")
        self.new = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.gone = torch.zeros(B, dtype=torch.bool, device="cuda")
        self.change()

    def change(self):
        self.new.copy_(torch.randint(0, 2 * self.T // self.B, (self.B,), dtype=torch.int32, device="cuda", generator=self.g))
        self.gone.copy_(torch.rand(self.B, device="cuda", generator=self.g) < 0.3)

    def run(self):
        return IU.page_plan_hip(self.lengths, self.new, self.table, self.ring, self.state, self.page, self.T, released=self.gone, inplace=True)

    def changed(self):
        return self.lengths, self.table, self.ring, self.state


class Store:
    def __init__(self, T, heads=4, kv=2, d=64):
        self.g, self.T = gen(T), T
        self.qkv = torch.randn(T, (heads + 2 * kv) * d, dtype=torch.float16, device="cuda", generator=self.g)
        self.kp, self.vp = torch.zeros(2, T // 16 + 2, kv, 16, d, dtype=torch.float16, device="cuda")
        self.cos, self.sin = torch.randn(2, 500, d // 2, dtype=torch.float16, device="cuda", generator=self.g)
        self.positions = torch.zeros(T, dtype=torch.int32, device="cuda")
        self.slots = torch.zeros(T, dtype=torch.int64, device="cuda")
        self.cut = heads * d, kv * d, kv * d
        self.change()

    def change(self):
        self.qkv.normal_(generator=self.g)
        self.positions.random_(0, 500, generator=self.g)
        self.slots.copy_(torch.randperm(self.T // 16 * 16 + 32, device="cuda", generator=self.g)[:self.T])

    def run(self):
        return IU.rope_store_paged_hip(*self.qkv.split(self.cut, 1), self.cos, self.sin, self.kp, self.vp, self.positions, self.slots,
                                       out=torch.empty(self.T, self.cut[0], dtype=torch.float16, device="cuda")),

    def changed(self):
        return self.kp, self.vp


class Attend:
    def __init__(self, B, longest, seed=1, heads=8, kv=2, d=128):
        self.g, self.B, self.longest, self.shape = gen(seed), B, longest, (heads, kv)
        self.max_pages = -(-longest // 16)
        pool = B * self.max_pages
        self.qkv = torch.randn(B, (heads + 2 * kv) * d, dtype=torch.float16, device="cuda", generator=self.g)
        self.kp, self.vp = torch.randn(2, pool, kv, 16, d, dtype=torch.float16, device="cuda", generator=self.g)
        self.cos, self.sin = torch.randn(2, longest, d // 2, dtype=torch.float16, device="cuda", generator=self.g) * 0.7
        self.table = torch.randperm(pool, device="cuda", generator=self.g).int().view(B, self.max_pages)
        self.lengths = torch.ones(B, dtype=torch.int32, device="cuda")
        self.slots = torch.zeros(B, dtype=torch.int64, device="cuda")
        self.change()

    def change(self):
        self.qkv.normal_(generator=self.g)
        self.lengths.random_(1, self.longest + 1, generator=self.g)
        at = self.lengths.long() - 1
        self.slots.copy_(self.table.gather(1, at[:, None] // 16)[:, 0].long() * 16 + at % 16)
        if self.B > 1:
            self.slots[int(torch.randint(self.B, (1,), device="cuda", generator=self.g))] = -1

    def run(self):
        return IU.attention_paged_hip(self.qkv, self.kp, self.vp, self.cos, self.sin, self.table, self.lengths, self.slots, *self.shape),

    def changed(self):
        return self.kp, self.vp


class Sample:
    def __init__(self, B, V, seed=2):
        self.g = gen(seed)
        self.x = torch.randn(B, V, dtype=torch.float16, device="cuda", generator=self.g)
        self.u, self.t, self.p, self.m = torch.rand(4, B, device="cuda", generator=self.g)
        self.k = torch.randint(0, V, (B,), dtype=torch.int32, device="cuda", generator=self.g)
        self.change()

    def change(self):
        self.x.normal_(generator=self.g)
        self.u.uniform_(generator=self.g)
        self.m.copy_(0.1 * torch.rand(self.m.shape, device="cuda", generator=self.g))

    def run(self):
        return IU.sample_hip(self.x, self.u, self.t, self.k, self.p, self.m),

    def changed(self):
        return ()


KINDS = {"plan": lambda: Plan(20, 40), "plan in two launches": lambda: Plan(40, 5000), "store": lambda: Store(33), "attention": lambda: Attend(3, 500), "attention in parts": lambda: Attend(3, 5000),
         "sample": lambda: Sample(5, 1000), "sample, long rows": lambda: Sample(3, 70001)}


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
    for _ in range(3):
        eager[1].change()
        cases[1].change()
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
    name = {Plan: "lengths", Store: "kp", Attend: "qkv", Sample: "x"}[type(case)]
    setattr(case, name, getattr(case, name).as_subclass(Other))
    assert same(case.run(), want.run()) and same(case.changed(), want.changed())
    assert len(calls) == 1
    for c in (case, want):
        c.change()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = case.run()
    for _ in range(3):
        graph.replay()
        assert same(got, want.run()) and same(case.changed(), want.changed())
        for c in (case, want):
            c.change()


@pytest.mark.parametrize("kind", [k for k in KINDS if "plan" not in k])
def test_again_and_again(kind):
    """The same call gives the same bits."""
    case = KINDS[kind]()
    first = [t.clone() for t in (*case.run(), *case.changed())]
    for _ in range(20):
        assert same((*case.run(), *case.changed()), first)
