"""logits_adjust_hip against the settings in 64 bits, token by token.

The bound of a result y: its rounding to fp16 (2^-11 |y|, or half of the smallest step, 2^-25), and four operations in fp32 (a quotient or product, a product, two or three sums),
each off by at most 2^-23 of the largest number on the way."""
import random

import numpy as np
import pytest
import torch

import tree_oracle as oracle
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def words(allowed, V):
    bits = np.zeros((len(allowed), -(-V // 32) * 32), dtype=np.uint8)
    for i, row in enumerate(allowed):
        bits[i, :V] = row
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy()).cuda()


class Case:
    """R rows of B requests, every setting on unless it is left out."""

    def __init__(self, R, V, B=None, history=40, width=None, biases=20, drafted=5, without=(), seed=0, masks=3, scale=3.0):
        rng, g = random.Random(seed + V), torch.Generator(device="cuda").manual_seed(seed + V)
        B = B or R
        self.R, self.V, self.B = R, V, B
        self.logits = (torch.randn(R, V, device="cuda", generator=g) * scale).half()
        token = lambda: rng.choice((rng.randrange(V), rng.randrange(min(V, 9)), -1, V, V + 5, 2 ** 31 - 1, -2 ** 31))        # noqa: E731
        number = lambda lo, hi: float(np.float32(rng.uniform(lo, hi)))     # noqa: E731
        width = width or history
        s = {"history": [[token() for _ in range(width)] for _ in range(B)], "history_lengths": [rng.randrange(history + 1) for _ in range(B)],
             "prompt_lengths": [rng.randrange(history + 1) for _ in range(B)], "repetition": [rng.choice((1.0, number(0.5, 2.0), 0.0, -3.0)) for _ in range(B)],
             "frequency": [rng.choice((0.0, number(-1, 2))) for _ in range(B)], "presence": [rng.choice((0.0, number(-1, 2))) for _ in range(B)],
             "drafted": [[rng.choice((-1, token())) for _ in range(drafted)] for _ in range(R)],
             "requests": [rng.randrange(B) for _ in range(R)] if B != R else list(range(R)),
             "bias_tokens": [[token() for _ in range(biases)] for _ in range(B)], "bias": [[number(-9, 9) for _ in range(biases)] for _ in range(B)],
             "allowed": [[rng.random() < (0.5, 0.95, 0.0)[m % 3] for _ in range(V)] for m in range(masks)], "allowed_rows": [rng.choice((-1, rng.randrange(masks), masks)) for _ in range(R)]}
        s.update({name: None for name in without})
        self.s = s

    def tensors(self):
        t = {}
        for name, v in self.s.items():
            if v is None:
                t[name] = None
            elif name == "allowed":
                t[name] = words(v, self.V)
            else:
                t[name] = torch.tensor(v, dtype=torch.float32 if name in ("repetition", "frequency", "presence", "bias") else torch.int32, device="cuda")
                if name in ("history", "drafted", "bias_tokens", "bias"):
                    t[name] = t[name].view(len(v), -1)
        return t

    def want(self):
        s, rows = self.s, []
        of = lambda name, b, none: none if s[name] is None else s[name][b]      # noqa: E731
        for r in range(self.R):
            b = r if s["requests"] is None else s["requests"][r]
            state = of("allowed_rows", r, r) if s["allowed"] is not None else -1
            allowed = s["allowed"][state] if s["allowed"] is not None and 0 <= state < len(s["allowed"]) else None
            x = self.logits[r].double().cpu().numpy()
            if not 0 <= b < self.B:
                rows.append(oracle.adjust(x, allowed=allowed))
                continue
            text = of("history", b, [])
            n = min(max(of("history_lengths", b, len(text)), 0), len(text))
            prompt = min(max(of("prompt_lengths", b, 0), 0), n)
            bias = list(zip(of("bias_tokens", b, []), of("bias", b, [])))
            counted = any(s[name] is not None for name in ("repetition", "frequency", "presence"))
            rows.append(oracle.adjust(x, text[:n] if counted else [], (text[prompt:n] + of("drafted", r, [])) if counted else [], of("repetition", b, 1.0), of("frequency", b, 0.0),
                                      of("presence", b, 0.0), bias, allowed))
        return torch.from_numpy(np.stack(rows)) if rows else torch.zeros(0, self.V, dtype=torch.float64)

    def check(self, **layout):
        print("logits adjust", self.R, self.V, self.B, [n for n, v in self.s.items() if v is not None], flush=True)
        settings, before, want = self.tensors(), self.logits.clone(), self.want()
        out = IU.logits_adjust_hip(self.logits, out=torch.empty_like(self.logits), **settings)
        assert torch.equal(self.logits.view(torch.int16), before.view(torch.int16))
        self.bounded(out, want)
        inplace = self.logits.clone()
        assert IU.logits_adjust_hip(inplace, **settings) is inplace and torch.equal(inplace.view(torch.int16), out.view(torch.int16))
        # rows that lie apart, on addresses that are no multiple of 16 bytes, with others' values between them
        wide = torch.full((self.R, self.V + 13), 7.0, dtype=torch.float16, device="cuda")
        part = wide[:, 3:3 + self.V]
        part.copy_(self.logits)
        IU.logits_adjust_hip(part, **settings)
        assert torch.equal(part.contiguous().view(torch.int16), out.view(torch.int16)) and bool((wide[:, :3] == 7).all()) and bool((wide[:, 3 + self.V:] == 7).all())
        return out

    def bounded(self, out, want):
        got, x = out.double().cpu(), self.logits.double().cpu()
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine].nan_to_num(nan=123), want[~fine].nan_to_num(nan=123)) and bool(torch.isfinite(got[fine]).all())
        biggest = 20 + 3 * x.nan_to_num(0, 0, 0).abs() + 2 * 60
        bound = 2.0 ** -11 * want.abs() + 2.0 ** -25 + 6 * 2.0 ** -23 * biggest
        assert bool(((got - want).abs() <= bound)[fine].all())


@pytest.mark.parametrize("V", [1, 7, 8, 31, 33, 100, 4095, 4096, 4097, 10338, 32000])
def test_vocabularies(V):
    Case(3, V).check()


@pytest.mark.parametrize("without", [
    ("allowed", "allowed_rows", "bias", "bias_tokens"), ("history", "history_lengths", "prompt_lengths", "repetition", "frequency", "presence", "drafted"),
    ("history", "history_lengths", "prompt_lengths", "repetition", "frequency", "presence", "drafted", "bias", "bias_tokens"), ("repetition",), ("frequency", "presence"),
    ("history_lengths",), ("prompt_lengths", "drafted"), ("history", "history_lengths", "prompt_lengths"), ("repetition", "frequency", "presence"),
    ("history", "history_lengths", "prompt_lengths", "repetition", "frequency", "presence", "drafted", "bias", "bias_tokens", "allowed", "allowed_rows")])
def test_settings_left_out(without):
    out = Case(4, 5000, without=without).check()
    if len(without) > 10:
        assert torch.equal(out, Case(4, 5000, without=without).logits)


@pytest.mark.parametrize("R,B", [(1, 1), (9, 4), (64, 3), (2, 300)])
def test_rows_of_requests(R, B):
    c = Case(R, 900, B=B)
    if R > 8:
        c.s["requests"][2], c.s["requests"][5], c.s["requests"][7] = -1, B, 2 ** 31 - 1          # rows of no request: the mask alone
    c.check()


def test_one_row_per_request_and_mask():
    Case(5, 700, without=("requests",)).check()
    Case(5, 700, masks=5, without=("requests", "allowed_rows")).check()


@pytest.mark.parametrize("history,width", [(1, 1), (511, 600), (513, 513), (5000, 5001)])
def test_lengths_of_the_text(history, width):
    Case(3, 600, history=history, width=width).check()
    c = Case(4, 600, history=history, width=width)
    c.s["history_lengths"], c.s["prompt_lengths"] = [0, width + 9, -4, width], [0, -3, 2, width + 1]
    c.check()


def test_many_of_one_token():
    """More of a token than 16 bits count."""
    c = Case(2, 50, history=70001, biases=1)
    c.s["history"], c.s["history_lengths"], c.s["prompt_lengths"] = [[3] * 70001, [3] * 70000 + [4]], [70001, 70001], [0, 70000]
    c.s["frequency"], c.s["presence"], c.s["repetition"] = [0.001, 0.5], [0.0, 0.25], [1.0, 1.5]
    c.logits.fill_(1.0)
    out = c.check()
    assert float(out[0, 3]) < -60


def test_of_several_entries_for_a_token_the_last_counts():
    c = Case(2, 5000, biases=700, without=("allowed", "allowed_rows"))
    for b in range(2):
        c.s["bias_tokens"][b] = [(i * 7) % 11 + 4090 * (i % 2) for i in range(700)]
    c.check()


def test_a_row_of_which_nothing_is_left():
    c = Case(3, 1000)
    c.s["allowed"], c.s["allowed_rows"] = [[False] * 1000, [i == 999 for i in range(1000)]], [0, 1, -1]
    out = c.check()
    assert bool((out[0] == float("-inf")).all()) and int(torch.isfinite(out[1]).sum()) == 1


def test_infinities_and_numbers_that_are_none():
    """In the logits they stay what they are, masked places are -inf whatever stood there; finite ones stay finite, infinite biases are added."""
    c = Case(3, 300, without=("allowed_rows",))
    c.logits[:, 0], c.logits[:, 1], c.logits[:, 2], c.logits[:, 3], c.logits[:, 4] = float("inf"), float("-inf"), float("nan"), 65504, -65504
    c.s["history"], c.s["history_lengths"], c.s["prompt_lengths"] = [list(range(40))] * 3, [40] * 3, [0] * 3
    c.s["repetition"], c.s["frequency"], c.s["presence"] = [0.001, 100.0, 1.0], [0.0, 2.0, 0.5], [0.0, -3.0, 0.0]
    c.s["bias_tokens"], c.s["bias"] = [[3, 4, 7, 8]] * 3, [[65504.0, -65504.0, float("inf"), float("-inf")], [-5.0, 5.0, float("-inf"), 3e38], [0.0, 0.0, 0.0, -3e38]]
    c.s["allowed"] = [[i not in (1, 2, 5) for i in range(300)], [i != 0 for i in range(300)], [True] * 300]
    out = c.check()
    assert float(out[0, 3]) == 65504 and float(out[0, 7]) == float("inf") and float(out[0, 2]) == float("-inf") and float(out[2, 8]) == -65504


def test_untouched_logits_keep_their_bits():
    c = Case(2, 70000, without=("bias", "bias_tokens", "allowed", "allowed_rows"), history=9)
    settings = c.tensors()
    out = IU.logits_adjust_hip(c.logits, out=torch.empty_like(c.logits), **settings)
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16).cuda().repeat(2, 1)
    same = IU.logits_adjust_hip(every, out=torch.empty_like(every), **{**settings, "history_lengths": torch.zeros_like(settings["history_lengths"]), "drafted": None})
    number = ~torch.isnan(every)
    assert torch.equal(same[number].view(torch.int16), every[number].view(torch.int16)) and bool(torch.isnan(same[~number]).all())
    assert int((out != c.logits).sum()) <= 2 * 14


def test_no_rows():
    assert IU.logits_adjust_hip(torch.zeros(0, 50, dtype=torch.float16, device="cuda")).shape == (0, 50)


def test_settings_of_no_width():
    """A text of no tokens, no drafted ones, no biases and no masks change nothing, beside others that do."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 5000, dtype=torch.float16, device="cuda", generator=g)
    i32 = dict(dtype=torch.int32, device="cuda")
    nothing = dict(history=torch.zeros(3, 0, **i32), history_lengths=torch.zeros(3, **i32), prompt_lengths=torch.zeros(3, **i32), repetition=torch.full((3,), 2.0, device="cuda"),
                   drafted=torch.zeros(3, 0, **i32), bias_tokens=torch.zeros(3, 0, **i32), bias=torch.zeros(3, 0, device="cuda"), allowed=torch.zeros(0, 157, **i32), allowed_rows=torch.full((3,), -1, **i32))
    for requests in (None, torch.tensor([2, 0, -1], **i32)):
        assert torch.equal(IU.logits_adjust_hip(x, out=torch.empty_like(x), requests=requests, **nothing), x)
    drafted = torch.tensor([[4], [-1], [4999]], **i32)
    y = IU.logits_adjust_hip(x, out=torch.empty_like(x), **{**nothing, "drafted": drafted})
    want = x.clone()
    for row, token in ((0, 4), (2, 4999)):
        v = x[row, token].double()
        want[row, token] = v / 2 if v > 0 else v * 2
    assert torch.equal(y, want)
