"""sample_hip against the definition in 64 bits, row by row.  The drawn index is a whole number and has to be equal: it is another one only where the random
number lies within about 1e-11 of the sum from a border."""
import numpy as np
import pytest
import torch

import paged_oracle as oracle
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def check(logits, u, **settings):
    """logits [B, V] fp16 on the device; u and the settings as lists."""
    B = logits.shape[0]
    dtypes = {"top_k": torch.int32}
    device = {k: torch.tensor(v, dtype=dtypes.get(k, torch.float32), device="cuda") for k, v in settings.items()}
    got = IU.sample_hip(logits, torch.tensor(u, dtype=torch.float32, device="cuda"), **device).tolist()
    x = logits.cpu().numpy()
    want = [oracle.sample(x[b], u[b], **{k: (np.float32(v[b]) if k != "top_k" else int(v[b])) for k, v in settings.items()}) for b in range(B)]
    assert got == want
    return got


def rows(B, V, seed, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, V, device="cuda", generator=g) * spread).half()


def numbers(B, seed, lo=0.0, hi=1.0):
    return (lo + (hi - lo) * np.random.RandomState(seed).rand(B)).astype(np.float32).tolist()


@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 7), (4, 8), (3, 511), (3, 513), (2, 8191), (40, 1000), (7, 32000), (3, 50257), (5, 128256), (2, 262144)])
@pytest.mark.parametrize("spread", [0.02, 1.0, 3.0])
def test_every_setting(B, V, spread):
    print(f"sample B={B} V={V} spread={spread}", flush=True)
    x = rows(B, V, V + B, spread)
    s = lambda i, lo, hi: numbers(B, 10 * i + B, lo, hi)          # noqa: E731
    k = lambda hi: np.random.RandomState(V).randint(1, hi, B).tolist()        # noqa: E731
    check(x, s(0, 0, 1))
    check(x, s(1, 0, 1), temperature=s(2, 0.1, 2))
    check(x, s(3, 0, 1), top_k=k(min(V, 60) + 1))
    check(x, s(4, 0, 1), top_k=k(V + 2), temperature=s(5, 0.1, 2))
    check(x, s(6, 0, 1), top_p=s(7, 0.01, 1))
    check(x, s(8, 0, 1), min_p=s(9, 0.0, 0.3))
    check(x, s(10, 0, 1), temperature=s(11, 0.3, 2), top_k=k(min(V, 1000) + 1), top_p=s(12, 0.3, 1), min_p=s(13, 0, 0.1))
    got = check(x, s(14, 0, 1), temperature=[0.0] * B)
    if V % 8 == 0:
        assert got == IU.argmax_hip(x).tolist()


@pytest.mark.parametrize("V", [9, 700, 40000])
def test_equal_values(V):
    """Few distinct values: the lowest indexes among equals stay, at the border of top-k and of top-p."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randint(-2, 3, (8, V), device="cuda", generator=g).half()
    x[0] = 1.5
    x[1] = -65504.0
    x[2, ::2] = 0.0
    x[2, 1::2] = -0.0
    u = numbers(8, 1)
    for k in (1, 2, V // 5 + 1, V // 2, V - 1, V, V + 1):
        check(x, u, top_k=[k] * 8)
        check(x, u, top_k=[k] * 8, top_p=[0.5] * 8)
    for p in (0.0, 0.001, 0.25, 0.5, 0.9, 0.999, 1.0, 1.5):
        check(x, u, top_p=[p] * 8)
    check(x, [0.0] * 8, top_k=[3] * 8)
    check(x, [1.0 - 2.0 ** -24] * 8, top_k=[3] * 8)


def test_values_without_weight():
    """-inf and NaN never come out, +inf takes all, a row of neither gives 0."""
    inf, nan = float("inf"), float("nan")
    x = rows(9, 1003, 4)
    x[0, 100:] = -inf
    x[1, :1000] = -inf
    x[2] = -inf
    x[3] = nan
    x[4, ::3] = nan
    x[5, 77], x[5, 900] = inf, inf
    x[6, :] = -inf
    x[6, 5] = -65504.0
    x[7, ::2] = -65504.0
    x[8, 40] = 60000.0
    for seed in range(3):
        u = numbers(9, seed)
        check(x, u)
        check(x, u, top_k=[50] * 9, top_p=[0.9] * 9, min_p=[0.01] * 9)
        check(x, u, top_k=[150] * 9)
        check(x, u, top_p=[0.99] * 9, temperature=[5.0] * 9)
        check(x, u, temperature=[0.0] * 9)


def test_settings_at_their_ends():
    x = rows(12, 3001, 8)
    u = [0.0, 1.0 - 2.0 ** -24, 0.5, float("nan"), -1.0, 1.0, 7.0, 0.25, 0.1, 0.9, 0.7, 0.3]
    nan, inf = float("nan"), float("inf")
    check(x, u)
    check(x, u, temperature=[0.0, -1.0, nan, 1e-30, 1e-5, 0.01, 100.0, 1e30, inf, 1.0, 2.0, 0.5])
    check(x, u, top_k=[0, -5, 1, 2, 3000, 3001, 3002, 2 ** 31 - 1, -2 ** 31, 10, 20, 30])
    check(x, u, top_p=[0.0, -1.0, 1e-30, 1.0, 2.0, inf, 0.5, 0.999999, 1.0 - 2.0 ** -24, 0.1, 0.2, 0.3])
    check(x, u, min_p=[0.0, -1.0, 1.0, 2.0, inf, 1e-30, 0.5, 0.9999, 0.1, 1e-3, 1e-6, 0.3])
    # (NaN: no top-p, no min-p)
    plain = check(x, u)
    f = lambda v: torch.full((12,), v, device="cuda")             # noqa: E731
    assert IU.sample_hip(x, torch.tensor(u, device="cuda"), top_p=f(nan), min_p=f(nan)).tolist() == plain


@pytest.mark.parametrize("ahead,ld", [(0, 1001), (1, 1001), (3, 1040), (7, 1007), (8, 1008)])
def test_rows_anywhere(ahead, ld):
    """Strides of any size, first values on any two bytes, NaN between the rows."""
    flat = torch.full((5 * ld + 16,), float("nan"), device="cuda", dtype=torch.float16)
    x = flat[ahead:ahead + 5 * ld].as_strided((5, 997), (ld, 1), ahead)
    x.copy_(rows(5, 997, ld))
    flat[ahead + 997:ahead + ld] = 60000.0 if ld > 997 else float("nan")
    if ahead:
        flat[:ahead] = 60000.0
    check(x, numbers(5, ahead))
    check(x, numbers(5, ahead + 1), top_k=[20] * 5, top_p=[0.8] * 5)


@pytest.mark.parametrize("temperature", [1e-30, 1e-4, 2e-3, 0.01, 0.1, 30.0, 1e30])
@pytest.mark.parametrize("size", [0.01, 3.0, 4000.0])
def test_weights_of_all_sizes(temperature, size):
    """Many tokens are kept, of which few, or all, weigh something: temperatures and values from one end to the other, with the least random numbers too."""
    B, V = 6, 9000
    x = (torch.randn(B, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)) * size).half()
    x[4] = -x[4].abs()
    u = [0.0, 1e-9, 0.3, 0.7, 0.0, 1.0 - 2.0 ** -24]
    for settings in (dict(top_k=3000), dict(top_p=0.999), dict(top_k=5000, top_p=0.99), dict(min_p=1e-30), {}):
        print(f"sample temperature={temperature} size={size} {settings}", flush=True)
        check(x, u, temperature=[temperature] * B, **{k: [v] * B for k, v in settings.items()})


def test_frequencies():
    """20000 draws of one row of 16 values: each count within six standard deviations of its weight's."""
    row = rows(1, 16, 2, 1.0)
    n = 20000
    g = torch.Generator(device="cuda").manual_seed(1)
    got = IU.sample_hip(row.expand(n, 16).contiguous(), torch.rand(n, device="cuda", generator=g))
    p = torch.softmax(row[0].double(), 0)
    count = torch.bincount(got, minlength=16)
    assert bool(((count - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all())


@pytest.mark.parametrize("V", [17, 600, 1025, 4000, 10338, 50257])
def test_top_k_at_the_ends_of_its_ways(V):
    """k around twice the spans, half the pieces of eight values, and the sizes of the lists."""
    spans, pieces = -(-V // 512), -(-V // 8)
    ks = sorted({k for n in (1, spans // 2, spans, 2 * spans, pieces // 2, 256, 512, 1024) for k in (n - 1, n, n + 1) if 1 <= k <= V})
    x = rows(len(ks), V, V)
    check(x, numbers(len(ks), 3), top_k=ks, temperature=[1.5] * len(ks))
    check(x, numbers(len(ks), 4), top_k=ks, top_p=[0.97] * len(ks))
    check(x.round(), numbers(len(ks), 5), top_k=ks, top_p=[0.9] * len(ks), temperature=[3.0] * len(ks))


@pytest.mark.parametrize("V", [3000, 33000])
def test_settings_together(V):
    """min-p drops tokens that top-p's sum still counts: every pair of settings, and all of them, with k below and above what a list holds."""
    x = rows(6, V, V, 2.0)
    u = numbers(6, V)
    for k in (3, 40, 260, 900, 1024, 1025, 2000):
        for t in (0.4, 1.0, 3.0):
            for p in (0.2, 0.9, 0.999):
                for m in (0.0, 0.01, 0.2):
                    check(x, u, temperature=[t] * 6, top_k=[k] * 6, top_p=[p] * 6, min_p=[m] * 6)
        check(x, u, top_k=[k] * 6, min_p=[0.02] * 6)
    for p in (0.2, 0.9, 0.999):
        check(x, u, top_p=[p] * 6, min_p=[0.02] * 6)
        check(x, u, top_p=[p] * 6, min_p=[0.0001] * 6, temperature=[2.0] * 6)
