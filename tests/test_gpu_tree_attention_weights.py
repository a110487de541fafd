"""The weights of attention_tree_hip's second product: held to 2^-22 of themselves, as the framework's other attentions of single tokens hold them.

Here all weights but one are the same number w, of which fp16 keeps (1 + r) w with r close to 2^-11, its worst; errors of single terms thus add up where those of random weights cancel.  Scores have one
product that is not zero, so what is left of their errors is the exponent's rounding (|15 + log2 w| * 2^-24) and the exponential's own: e = 2^-20 of a weight is allowed.  Two fp16 terms: 2^-22.  The sums'
roundings in fp32, chains of at most 2^9 steps above and below the line: 2^-14 in all."""
import numpy as np
import pytest
import torch

from test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu

QUERY = 2.0
BUILDS = [(8, 2, 4), (8, 2, 8), (8, 2, 16), (8, 2, 32), (16, 2, 64)]       # heads, KV heads, nodes: 16, 32, 64, 128, 512 rows of a KV head


def weight_of(key, d):
    return np.exp(QUERY * np.float64(key) / d ** 0.5)


def key_of(d):
    """The key, of those that put the weight at 0.5 to 0.6 of the largest, whose weight fp16 rounds up the farthest (the largest as 2^15)."""
    keys = -np.arange(2.0, 4.0, 2.0 ** -9).astype(np.float16)
    weights = weight_of(keys, d)
    up = ((weights * 2.0 ** 15).astype(np.float16).astype(np.float64) / 2.0 ** 15 - weights) / weights
    up[(weights < 0.5) | (weights > 0.6)] = 0
    best = int(up.argmax())
    assert up[best] > 0.8 * 2.0 ** -11
    return float(keys[best])


def case_of(heads, kv, nodes, d, held):
    c = Case(heads, kv, d, 16, [held], [nodes], kind="any")
    c.masks = [-1] * nodes                        # every node sees all
    c.q.zero_()
    c.q.view(nodes, heads, d)[..., 0] = QUERY
    for row in c.rows[0]:
        c.kpages[row].zero_()
        c.kpages[row, :, :, 0] = key_of(d)
    c.kpages[c.rows[0][0], :, 0, 0] = 0.0         # position 0 has the weight 1
    return c


@pytest.mark.parametrize("heads,kv,nodes", BUILDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("held", [31, 5000])
@pytest.mark.parametrize("value", [65504.0, -65504.0, 1.0])
def test_what_all_positions_have_comes_out_as_it_is(heads, kv, nodes, d, held, value):
    """The errors of a weight and of the exponentials stand above and below the line; a result is off by 2^-14 + 2^-21 at most before it is rounded, and fp16's half step at these values is 2^-12: it is the value, and
    no infinity."""
    c = case_of(heads, kv, nodes, d, held)
    for row in c.rows[0]:
        c.vpages[row] = value
    out = c.run()
    assert bool((out == value).all()), (out.min(), out.max())


@pytest.mark.parametrize("heads,kv,nodes", BUILDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("held", [31, 5000])
def test_what_cancels_is_not_lost(heads, kv, nodes, d, held):
    """Position 0 takes away what the others have together: little is left of sums that are far larger."""
    c = case_of(heads, kv, nodes, d, held)
    w, others = weight_of(key_of(d), d), held + nodes - 1
    value = (1 + torch.arange(kv * d, device="cuda").view(kv, 1, d) / (kv * d)).half()
    for row in c.rows[0]:
        c.vpages[row] = value
    first = (-others * w * value.double()).half()
    c.vpages[c.rows[0][0], :, :1] = first
    want = (first.double() + others * w * value.double()) / (1 + others * w)
    spread = (first.double().abs() + others * w * value.double()) / (1 + others * w)
    bound = 2.0 ** -11 * want.abs() + 2.0 ** -25 + (2.0 ** -14 + 2.0 ** -21 + 2 * 2.0 ** -20) * spread
    off = (c.run().view(nodes, kv, heads // kv, d).double() - want.view(1, kv, 1, d)).abs()
    print(f"  worst {float((off / bound.view(1, kv, 1, d)).max()):.3f} of the bound", flush=True)
    assert bool((off <= bound.view(1, kv, 1, d)).all())
