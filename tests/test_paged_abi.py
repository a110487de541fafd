"""What the entry points for requests of unequal lengths refuse, on the CPU: every refusal comes before anything is launched."""
import ctypes
import os

import pytest
import torch

from bitstack_amd import _lib
from bitstack_amd.utils import inference_utils as IU

NUL, ONE = ctypes.c_void_p(0), ctypes.c_void_p(4096)          # (never dereferenced on these paths)
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


PLAN = dict(lengths=ONE, new=ONE, released=NUL, table=ONE, ring=ONE, state=ONE, lengths_out=ONE, state_out=ONE, granted=ONE, starts=ONE, positions=ONE, slots=ONE, row_slots=NUL,
            B=4, T=5000, page=16, max_pages=8, pool=100, ws=ONE, ws_bytes=1 << 20, stream=NUL)
STORE = dict(q=ONE, ldq=512, q_out=NUL, ldq_out=0, k=ONE, v=ONE, ldkv=256, cos=ONE, sin=ONE, positions=ONE, slots=ONE, kpages=ONE, vpages=ONE, T=4, heads=4, kv_heads=2,
             d=128, max_pos=100, page=16, pool=100, stream=NUL)
ATTEND = dict(qkv=ONE, ld=1024, kpages=ONE, vpages=ONE, cos=ONE, sin=ONE, table=ONE, lengths=ONE, slots=ONE, out=ONE, B=4, heads=4, kv_heads=2, d=128, max_pos=5000, page=16,
              max_pages=300, pool=100, ws=ONE, ws_bytes=1 << 30, stream=NUL)
SAMPLE = dict(logits=ONE, ld=1000, uniform=ONE, temperature=NUL, top_k=NUL, top_p=NUL, min_p=NUL, out=ONE, B=4, V=1000, ws=ONE, ws_bytes=1 << 20, stream=NUL)
ODD = ctypes.c_void_p(4097)
EIGHT = ctypes.c_void_p(4104)


def test_plan(L):
    refused = lambda **c: call(L.bs_page_plan, PLAN, **c)                 # noqa: E731
    for name in ("lengths", "new", "table", "ring", "state", "lengths_out", "state_out", "granted", "starts", "positions", "slots"):
        assert refused(**{name: NUL}) == NULLS, name
        assert refused(**{name: ODD}) == ALIGN, name
    assert refused(slots=ctypes.c_void_p(4100)) == refused(row_slots=ctypes.c_void_p(4100)) == ALIGN
    for change in ({"B": -1}, {"B": 65537}, {"T": -1}, {"T": (1 << 30) + 1}, {"page": 8}, {"page": 24}, {"page": 2048}, {"page": 0}, {"page": -16}, {"max_pages": 0},
                   {"max_pages": (1 << 24) + 1}, {"pool": 0}, {"pool": 1 << 27}):
        assert refused(**change) == SHAPE, change
    assert refused(ws=NUL) == refused(ws_bytes=10) == refused(ws=EIGHT) == WORKSPACE
    assert L.bs_page_plan_workspace_bytes(4, 5000) > 0 == L.bs_page_plan_workspace_bytes(64, 64)
    assert L.bs_page_plan_workspace_bytes(-1, 4) == L.bs_page_plan_workspace_bytes(4, -1) == SHAPE


def test_store(L):
    refused = lambda **c: call(L.bs_rope_store_paged_f16, STORE, **c)     # noqa: E731
    for name in ("k", "v", "cos", "sin", "positions", "slots", "kpages", "vpages"):
        assert refused(**{name: NUL}) == NULLS, name
        assert refused(**{name: ODD}) == ALIGN, name
    assert refused(q=ODD) == refused(q_out=ODD, ldq_out=512) == refused(positions=ctypes.c_void_p(4098)) == refused(slots=ctypes.c_void_p(4100)) == ALIGN
    for change in ({"T": -1}, {"d": 96}, {"d": 256}, {"kv_heads": 0}, {"heads": 0}, {"max_pos": 0}, {"page": 17}, {"pool": 0}, {"pool": 1 << 28}, {"ldq": 511}, {"ldkv": 255},
                   {"q_out": EIGHT, "ldq_out": 511}, {"q_out": ONE, "ldq_out": 520}, {"q": NUL, "q_out": ONE, "ldq_out": 512}, {"kv_heads": 1 << 30}):
        assert refused(**change) == SHAPE, change
    assert refused(T=0) == refused(T=0, q=NUL, heads=0) == 0


def test_attention(L):
    refused = lambda **c: call(L.bs_attention_paged_f16, ATTEND, **c)     # noqa: E731
    for name in ("qkv", "kpages", "vpages", "cos", "sin", "table", "lengths", "slots", "out"):
        assert refused(**{name: NUL}) == NULLS, name
        assert refused(**{name: ODD}) == ALIGN, name
    assert refused(kpages=EIGHT) == refused(vpages=EIGHT) == refused(slots=ctypes.c_void_p(4100)) == ALIGN
    for change in ({"B": -1}, {"B": 65537}, {"heads": 0}, {"kv_heads": 0}, {"heads": 5}, {"d": 96}, {"d": 32}, {"page": 48}, {"page": 8}, {"max_pages": 0}, {"max_pos": 0},
                   {"pool": 0}, {"pool": 1 << 27}, {"ld": 1023}, {"max_pages": 1 << 27}, {"B": 65536, "max_pages": 1 << 20}, {"B": 65536, "heads": 128, "max_pages": 4, "ld": 1 << 20}):
        assert refused(**change) == SHAPE, change
    assert refused(ws=NUL) == refused(ws_bytes=100) == refused(ws=EIGHT) == WORKSPACE
    assert refused(B=0) == 0
    bytes_of = L.bs_attention_paged_workspace_bytes
    assert bytes_of(0, 4, 2, 128, 16, 300) == 0 == bytes_of(4, 4, 2, 128, 16, 4)
    assert bytes_of(4, 5, 2, 128, 16, 300) == bytes_of(4, 4, 2, 100, 16, 300) == bytes_of(4, 4, 2, 128, 20, 300) == SHAPE


def test_sample(L):
    refused = lambda **c: call(L.bs_sample_f16, SAMPLE, **c)              # noqa: E731
    for name in ("logits", "uniform", "out"):
        assert refused(**{name: NUL}) == NULLS, name
    for name in ("logits", "uniform", "temperature", "top_k", "top_p", "min_p", "out"):
        assert refused(**{name: ODD}) == ALIGN, name
    assert refused(out=ctypes.c_void_p(4100)) == refused(top_k=ctypes.c_void_p(4098)) == ALIGN
    for change in ({"B": -1}, {"B": (1 << 20) + 1}, {"V": 0}, {"V": (1 << 18) + 1}, {"ld": 999}, {"ld": -1000}, {"B": 1 << 20, "V": 9000, "ld": 9000}):
        assert refused(**change) == SHAPE, change
    assert refused(ws=NUL) == refused(ws_bytes=10) == refused(ws=EIGHT) == WORKSPACE
    assert L.bs_sample_workspace_bytes(4, 0) == L.bs_sample_workspace_bytes(-1, 10) == SHAPE and L.bs_sample_workspace_bytes(0, 10) == 0
    assert refused(B=0) == 0


def test_tensors_on_the_cpu_are_refused():
    i32 = torch.zeros(2, dtype=torch.int32)
    half = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="HIP device"):
        IU.page_plan_hip(i32, i32, i32.view(2, 1), i32, i32, 16, 4)
    with pytest.raises(RuntimeError, match="HIP device"):
        IU.rope_store_paged_hip(None, half, half, half, half, half, half, i32, i32)
    with pytest.raises(RuntimeError, match="HIP device"):
        IU.attention_paged_hip(half, half, half, half, half, i32, i32, i32, 1, 1)
    with pytest.raises(RuntimeError, match="HIP device"):
        IU.sample_hip(half.view(2, -1), torch.zeros(2))
