"""sample_hip on rows whose frequent tokens stand together: vocabularies are ordered by frequency, so that what top-p keeps lies in front, or in two places with
nothing between them.  Against the definition in 64 bits; tokens are whole numbers and have to be equal."""
import numpy as np
import pytest
import torch

import paged_oracle as oracle
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu

# both ends, and enough between them that every part of a row is drawn from
NUMBERS = [0.0, 1e-6, 0.03, 0.1, 0.2, 0.3, 0.4, 0.5, 0.6, 0.7, 0.8, 0.9, 0.95, 0.99, 0.9999, 1.0 - 2.0 ** -24]


def check(x, **settings):
    """One row x (fp16, [V]) with every random number, one setting each for all of them."""
    n = len(NUMBERS)
    u = torch.tensor(NUMBERS, dtype=torch.float32, device="cuda")
    device = {k: torch.full((n,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda") for k, v in settings.items()}
    got = IU.sample_hip(x.expand(n, -1).contiguous(), u, **device).tolist()
    row = x.cpu().numpy()
    assert got == [oracle.sample(row, v, **settings) for v in NUMBERS], settings


@pytest.mark.parametrize("V", [128256, 50257, 33001])
@pytest.mark.parametrize("turned", [False, True])
def test_few_large_ones_far_from_many(V, turned):
    """2000 equal tokens at one end, ten larger ones at the other, of all others every one weighs little and none stays."""
    x = torch.full((V,), -3.0, dtype=torch.float16, device="cuda")
    x[:2000], x[-10:] = 0.0, 0.5
    x = x.flip(0) if turned else x
    for p in (0.05, 0.15, 0.18, 0.22):
        check(x, top_p=p)
        check(x, top_p=p, min_p=0.01)


@pytest.mark.parametrize("V", [128256, 40000])
@pytest.mark.parametrize("fall", [-12.0, -6.0, -4.0, 4.0, 6.0, 12.0])
def test_rows_with_a_slope(V, fall):
    """Normal logits that fall (or rise) along the vocabulary."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(V, device="cuda", generator=g) * 2.0 - fall * torch.arange(V, device="cuda") / V).half()
    for settings in (dict(top_p=0.2), dict(top_p=0.5), dict(top_p=0.8), dict(top_p=0.97), dict(top_p=0.9, temperature=1.5), dict(top_p=0.5, min_p=1e-4),
                     dict(top_k=3000, top_p=0.6), dict(top_k=5000), dict(top_p=0.999, temperature=0.3)):
        check(x, **settings)


@pytest.mark.parametrize("V", [128256, 20011])
@pytest.mark.parametrize("ends", [(0.0, 0.02, 0.5, 0.55), (0.3, 0.4, 0.9, 1.0), (0.0, 0.1, 0.98, 1.0)])
def test_two_places(V, ends):
    """What stays is equal tokens (ties at the border) in two places, and the larger ones in one of them; nothing stays between, which weighs most of the sum."""
    a, b, c, d = (int(V * e) for e in ends)
    g = torch.Generator(device="cuda").manual_seed(a + d)
    low = torch.rand(V, device="cuda", generator=g) - 2.5
    for first, second in ((1.0, 1.5), (1.5, 1.0), (1.0, 1.0)):
        x = low.clone()
        x[a:b], x[c:d] = first, second
        x = x.half()
        w = np.exp(x.double().cpu().numpy() - max(first, second))
        both = (w[a:b].sum() + w[c:d].sum()) / w.sum()
        for part in (0.3, 0.6, 0.9, 0.999):
            check(x, top_p=float(np.float32(both * part)))
