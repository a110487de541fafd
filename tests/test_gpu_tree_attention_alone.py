"""A NaN in a query or a key, an infinity in a value: rows and heads whose products it is in none of keep every bit, the rest of its own rows what 64 bits give."""
import pytest
import torch

from test_gpu_tree_attention import NAN, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", ["q", "key", "value"])
@pytest.mark.parametrize("held,counts", [([300, 40], [6, 3]), ([3000, 40], [64, 3]), ([700, 90], [16, 30]), ([60, 40], [4, 2])])
def test_others_keep_their_bits(where, held, counts, d):
    c = Case(4, 2, d, 16, held, counts)
    want = c.run().view(-1, 4, d)
    changed = torch.zeros(want.shape[0], 4, dtype=torch.bool, device="cuda")
    if where == "q":
        c.q[1, d + 2] = NAN
        changed[1, 1] = True
    elif where == "key":
        c.kpages[c.rows[0][2], 0, 5, 9] = NAN
        changed[:counts[0], :2] = True
    else:
        c.vpages[c.rows[0][2], 1, 5, 9] = float("inf")
        changed[:counts[0], 2:] = True
    out = c.run().view(-1, 4, d)
    assert torch.equal(out[~changed].view(torch.int16), want[~changed].view(torch.int16))
    if where != "value":
        assert bool(torch.isnan(out[changed]).all())
        return
    assert bool((out[changed][:, 9] == float("inf")).all())
    # computed again in fp32: two roundings to fp16 of numbers that are next to one another (2^-11 of the value each, 2^-25 below fp16's full numbers), and twice the sums' 2^-13 of what is summed
    rest = [i for i in range(d) if i != 9]
    a, b = out[changed][:, rest].double(), want[changed][:, rest].double()
    largest = c.vpages[c.rows[0], 1].nan_to_num(0.0, 0.0, 0.0).abs().max().double()
    assert bool(((a - b).abs() <= 2.0 ** -10 * a.abs() + 2.0 ** -24 + 2.0 ** -12 * largest).all())
