"""Caches and logits of more values than 32 bits count: the operators for drafted trees, forked rows and settings on logits at their last places."""
import pytest
import torch

from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu

LAYERS, POOL, KV, PAGE, D = 2, 33000, 8, 64, 128          # (a layer has 2.16e9 values)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def i64(v):
    return torch.tensor(v, dtype=torch.int64, device="cuda")


@pytest.fixture(scope="module", autouse=True)
def memory_goes_back():
    """(What later tests keep would else be cut from these tensors' memory, which then stays.)"""
    yield
    torch.cuda.empty_cache()


@pytest.fixture(scope="module")
def caches():
    pages = torch.zeros(2, LAYERS, POOL, KV, PAGE, D, dtype=torch.float16, device="cuda")
    assert pages[0, 0].numel() > 2 ** 31
    yield pages


def fill(caches, used):
    caches.zero_()
    for p in used:
        caches[:, :, p].normal_(generator=torch.Generator(device="cuda").manual_seed(p))
    return {p: caches[:, :, p].clone() for p in used}


def check(caches, want):
    for p, t in want.items():
        assert torch.equal(caches[:, :, p], t), p
    assert sum(int(torch.count_nonzero(caches[i, L])) for i in range(2) for L in range(LAYERS)) == sum(int(torch.count_nonzero(t)) for t in want.values())


def test_accept(caches):
    """Nodes at 62 .. 65 of a request: the path 0, 2, 3 moves across a page's end."""
    first, second = POOL - 1, POOL - 2
    want = fill(caches, (first, second, 5))
    ring, state = i32([0] * POOL), i32([0, 0])
    slots = [first * PAGE + 62, first * PAGE + 63, second * PAGE, second * PAGE + 1]
    done = IU.tree_accept_hip(i64([7, 1, 2, 3]), i32([-1, 0, 0, 2]), i64([2, 9, 3, 4]), i64(slots), i32([66]), i32([4]), i32([0, 4]), i32([[first, second]]), ring, state, *caches, nodes=4)
    assert done.path.tolist() == [[0, 2, 3, -1]] and done.lengths.tolist() == [65] and done.token.tolist() == [4]
    old = {p: t.clone() for p, t in want.items()}
    want[first][:, :, :, 63] = old[second][:, :, :, 0]
    want[second][:, :, :, 0] = old[second][:, :, :, 1]
    check(caches, want)


def test_fork(caches):
    """The last page, not full, to a new one."""
    whole, last, fresh = POOL - 1, POOL - 2, POOL - 4
    want = fill(caches, (whole, last, 5))
    ring, state, shares, table = i32([fresh] + [0] * (POOL - 1)), i32([0, 1]), torch.zeros(POOL, dtype=torch.int32, device="cuda"), i32([[whole, last], [0, 0]])
    done = IU.page_fork_hip(i32([0, 0]), i32([70, 0]), table, ring, state, shares, *caches)
    assert done.granted.tolist() == [1, 1] and done.lengths.tolist() == [70, 70] and table.tolist() == [[whole, last], [whole, fresh]] and int(shares[whole]) == 1 == int(shares.sum())
    want[fresh] = torch.zeros_like(want[last])
    want[fresh][:, :, :, :6] = want[last][:, :, :, :6]
    check(caches, want)


def test_adjust():
    """Rows behind the first 2^31 logits are what they are by themselves."""
    R, V = 16500, 131072
    x = torch.empty(R, V, dtype=torch.float16, device="cuda")
    assert x.numel() > 2 ** 31
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    rows = [0, 16383, 16384, R - 1]
    g = torch.Generator(device="cuda").manual_seed(2)
    settings = dict(history=torch.randint(0, V, (2, 5000), dtype=torch.int32, device="cuda", generator=g), repetition=torch.tensor([1.3, 0.8], device="cuda"), presence=torch.tensor([0.5, 0.0], device="cuda"),
                    bias_tokens=torch.randint(0, V, (2, 30), dtype=torch.int32, device="cuda", generator=g), bias=torch.randn(2, 30, device="cuda", generator=g),
                    allowed=torch.randint(-2 ** 31, 2 ** 31 - 1, (2, V // 32), dtype=torch.int32, device="cuda", generator=g))
    requests, states = torch.full((2, R), -1, dtype=torch.int32, device="cuda")
    requests[rows], states[rows] = i32([0, 1, 0, 1]), i32([1, 0, 0, -1])
    want = IU.logits_adjust_hip(x[rows], requests=requests[rows], allowed_rows=states[rows], **settings)
    untouched = x[rows[2] + 1:rows[2] + 3].clone()
    IU.logits_adjust_hip(x, requests=requests, allowed_rows=states, **settings)
    assert torch.equal(x[rows], want) and torch.equal(x[rows[2] + 1:rows[2] + 3], untouched)
    assert bool((want[0] == -torch.inf).any()) and not bool((want[3] == -torch.inf).any())
