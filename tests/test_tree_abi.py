"""What the entry points for drafted trees, forked rows and settings on logits refuse, on the CPU: every refusal comes before anything is launched."""
import ctypes
import os

import pytest
import torch

from bitstack_amd import _lib
from bitstack_amd.utils import inference_utils as IU

NUL, ONE = ctypes.c_void_p(0), ctypes.c_void_p(4096)          # (never dereferenced on these paths)
ODD, TWO, FOUR, EIGHT = (ctypes.c_void_p(4096 + n) for n in (1, 2, 4, 8))
NULLS, SHAPE, ALIGN, WORKSPACE = -1, -2, -4, -5


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build(force=False)
    return _lib.lib()


def call(fn, spec, **changed):
    args = dict(spec, **changed)
    assert set(args) == set(spec), changed
    return fn(*args.values())


PLAN = dict(parents=ONE, lengths=ONE, granted=ONE, starts=ONE, positions=ONE, masks=ONE, B=4, T=20, stream=NUL)
ATTEND = dict(q=ONE, ldq=512, kpages=ONE, vpages=ONE, table=ONE, lengths=ONE, granted=ONE, starts=ONE, masks=ONE, out=ONE, B=4, T=20, nodes=8, heads=4, kv_heads=2, d=128, page=16,
              max_pages=300, pool=100, ws=ONE, ws_bytes=1 << 40, stream=NUL)
ACCEPT = dict(tokens=ONE, parents=ONE, targets=ONE, slots=ONE, lengths=ONE, granted=ONE, starts=ONE, table=ONE, ring=ONE, state=ONE, kpages=ONE, vpages=ONE, lengths_out=ONE, state_out=ONE,
              accepted=ONE, path=ONE, token=ONE, B=4, T=20, nodes=8, layers=2, kv_heads=2, d=128, page=16, max_pages=8, pool=100, ws=ONE, ws_bytes=1 << 20, stream=NUL)
FORK = dict(source=ONE, lengths=ONE, table=ONE, ring=ONE, state=ONE, shares=ONE, kpages=ONE, vpages=ONE, lengths_out=ONE, state_out=ONE, granted=ONE, B=4, layers=2, kv_heads=2, d=128, page=16,
            max_pages=8, pool=100, ws=ONE, ws_bytes=1 << 20, stream=NUL)
ADJUST = dict(logits=ONE, ld=1000, out=ONE, ld_out=1000, requests=ONE, history=ONE, width=50, history_lengths=ONE, prompt_lengths=ONE, repetition=ONE, frequency=ONE, presence=ONE, drafted=ONE,
              drafted_width=5, bias_tokens=ONE, bias=ONE, biases=9, allowed=ONE, masks=3, allowed_rows=ONE, R=4, V=1000, B=2, stream=NUL)


def test_plan(L):
    refused = lambda **c: call(L.bs_tree_plan, PLAN, **c)                 # noqa: E731
    for name in ("parents", "lengths", "granted", "starts", "positions", "masks"):
        assert refused(**{name: NUL}) == NULLS and refused(**{name: ODD}) == refused(**{name: TWO}) == ALIGN, name
    assert refused(masks=FOUR) == ALIGN
    for change in ({"B": -1}, {"B": 65537}, {"T": -1}, {"T": (1 << 30) + 1}):
        assert refused(**change) == SHAPE, change
    assert refused(T=0) == 0


def test_attention(L):
    refused = lambda **c: call(L.bs_attention_tree_f16, ATTEND, **c)      # noqa: E731
    for name in ("q", "kpages", "vpages", "table", "lengths", "granted", "starts", "masks", "out"):
        assert refused(**{name: NUL}) == NULLS and refused(**{name: ODD}) == ALIGN, name
    assert refused(kpages=EIGHT) == refused(vpages=EIGHT) == refused(masks=FOUR) == refused(table=TWO) == ALIGN
    for change in ({"B": -1}, {"B": 65537}, {"T": -1}, {"T": 1 << 21}, {"nodes": 0}, {"nodes": 65}, {"heads": 0}, {"kv_heads": 0}, {"heads": 5}, {"d": 96}, {"d": 32}, {"page": 48}, {"page": 8},
                   {"max_pages": 0}, {"pool": 0}, {"pool": 1 << 27}, {"ldq": 511}, {"max_pages": 1 << 27}, {"B": 65536, "max_pages": 1 << 20}):
        assert refused(**change) == SHAPE, change
    assert refused(ws=NUL) == refused(ws_bytes=100) == refused(ws=EIGHT) == WORKSPACE
    assert refused(T=0) == 0
    bytes_of = L.bs_attention_tree_workspace_bytes
    assert bytes_of(4, 20, 8, 4, 2, 128, 16, 300) > 0 == bytes_of(4, 20, 8, 4, 2, 128, 16, 4) == bytes_of(0, 20, 8, 4, 2, 128, 16, 300) == bytes_of(4, 0, 8, 4, 2, 128, 16, 300)
    assert bytes_of(4, 20, 8, 5, 2, 128, 16, 300) == bytes_of(4, 20, 65, 4, 2, 128, 16, 300) == bytes_of(4, 20, 8, 4, 2, 100, 16, 300) == SHAPE


def test_accept(L):
    refused = lambda **c: call(L.bs_tree_accept_f16, ACCEPT, **c)         # noqa: E731
    pointers = [name for name in ACCEPT if name not in ("B", "T", "nodes", "layers", "kv_heads", "d", "page", "max_pages", "pool", "ws", "ws_bytes", "stream")]
    for name in pointers:
        assert refused(**{name: NUL}) == NULLS and refused(**{name: ODD}) == ALIGN, name
    for name in ("tokens", "targets", "slots", "token", "kpages", "vpages"):
        assert refused(**{name: FOUR}) == ALIGN, name
    for change in ({"B": -1}, {"B": 65537}, {"T": -1}, {"T": (1 << 30) + 1}, {"nodes": 0}, {"nodes": 65}, {"layers": 0}, {"kv_heads": 0}, {"d": 0}, {"d": 60}, {"page": 24}, {"max_pages": 0},
                   {"B": 65536, "max_pages": 1 << 16}, {"pool": 0}, {"pool": 1 << 27}, {"layers": 1 << 20}, {"kv_heads": 1 << 21}, {"layers": 1 << 30, "kv_heads": 1 << 20, "d": 1 << 20}):
        assert refused(**change) == SHAPE, change
    assert refused(ws=NUL) == refused(ws_bytes=10) == refused(ws=EIGHT) == WORKSPACE
    assert L.bs_tree_accept_workspace_bytes(-1) == L.bs_tree_accept_workspace_bytes(65537) == SHAPE


def test_fork(L):
    refused = lambda **c: call(L.bs_page_fork_f16, FORK, **c)             # noqa: E731
    for name in ("source", "lengths", "table", "ring", "state", "shares", "kpages", "vpages", "lengths_out", "state_out", "granted"):
        assert refused(**{name: NUL}) == NULLS and refused(**{name: ODD}) == ALIGN, name
    assert refused(kpages=EIGHT) == refused(vpages=EIGHT) == ALIGN
    for change in ({"B": -1}, {"B": 65537}, {"layers": 0}, {"kv_heads": 0}, {"d": 4}, {"d": 12}, {"page": 0}, {"max_pages": 0}, {"max_pages": (1 << 24) + 1}, {"B": 65536, "max_pages": 1 << 16},
                   {"pool": 0}, {"pool": 1 << 27}, {"layers": 1 << 20}):
        assert refused(**change) == SHAPE, change
    assert refused(ws=NUL) == refused(ws_bytes=10) == refused(ws=EIGHT) == WORKSPACE
    assert L.bs_page_fork_workspace_bytes(-1, 8, 100) == L.bs_page_fork_workspace_bytes(4, 0, 100) == L.bs_page_fork_workspace_bytes(4, 8, 0) == SHAPE


def test_adjust(L):
    refused = lambda **c: call(L.bs_logits_adjust_f16, ADJUST, **c)       # noqa: E731
    assert refused(logits=NUL) == refused(out=NUL) == NULLS
    for name in ("logits", "out", "requests", "history", "history_lengths", "prompt_lengths", "repetition", "frequency", "presence", "drafted", "bias_tokens", "bias", "allowed", "allowed_rows"):
        assert refused(**{name: ODD}) == ALIGN, name
    assert refused(history=TWO) == refused(bias=TWO) == ALIGN
    for change in ({"R": -1}, {"R": (1 << 20) + 1}, {"V": 0}, {"V": (1 << 18) + 1}, {"ld": 999}, {"ld_out": 999}, {"B": -1}, {"width": -1}, {"drafted_width": -1}, {"biases": -1}, {"masks": -1}, {"width": (1 << 30) + 1}, {"drafted_width": (1 << 31) - 1}, {"biases": (1 << 31) - 1},
                   {"history": NUL}, {"bias": NUL}, {"bias_tokens": NUL}, {"allowed": NUL}, {"allowed_rows": NUL}, {"requests": NUL}, {"ld_out": 1001}, {"R": 1 << 20, "V": 9000, "ld": 9000, "ld_out": 9000}):
        assert refused(**change) == SHAPE, change
    assert refused(R=0) == 0


def test_tensors_on_the_cpu_are_refused():
    i32, i64 = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    half = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    for fn in (lambda: IU.tree_plan_hip(i32, i32, i32, i32), lambda: IU.attention_tree_hip(half.view(2, -1), half, half, i32.view(2, 1), i32, i32, i32, i64),
               lambda: IU.tree_accept_hip(i64, i32, i64, i64, i32, i32, i32, i32.view(2, 1), i32, i32, half, half), lambda: IU.page_fork_hip(i32, i32, i32.view(2, 1), i32, i32, i32, half, half),
               lambda: IU.logits_adjust_hip(half.view(2, -1))):
        with pytest.raises(RuntimeError, match="HIP device"):
            fn()
