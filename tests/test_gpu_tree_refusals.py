"""What the Python entry points for drafted trees, forked rows and settings on logits refuse: types, shapes and layouts that the kernels do not take, before anything is
launched."""
import pytest
import torch

from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32, device="cuda")


def i64(*shape):
    return torch.zeros(*shape, dtype=torch.int64, device="cuda")


def f16(*shape):
    return torch.zeros(*shape, dtype=torch.float16, device="cuda")


def f32(*shape):
    return torch.zeros(*shape, device="cuda")


def refuse(fn, good, cases):
    fn(**good)
    for change in cases:
        with pytest.raises((ValueError, RuntimeError)):
            fn(**{**good, **change})
            pytest.fail(str({name: getattr(t, "shape", t) for name, t in change.items()}))


def test_plan():
    good = dict(parents=i32(5), lengths=i32(3), granted=i32(3), starts=i32(4))
    refuse(IU.tree_plan_hip, good, [{"parents": i32(5).long()}, {"parents": i32(5, 1)}, {"parents": i32(10)[::2]}, {"lengths": i32(3).long()}, {"lengths": i32(2)}, {"granted": i32(4)}, {"granted": f32(3)},
                                    {"starts": i32(3)}, {"starts": i64(4)}, {"lengths": torch.zeros(3, dtype=torch.int32)}])


def test_attention():
    good = dict(q=f16(5, 256), kpages=f16(4, 1, 16, 128), vpages=f16(4, 1, 16, 128), block_table=i32(3, 4), lengths=i32(3), granted=i32(3), starts=i32(4), masks=i64(5), nodes=8, out=None)
    refuse(IU.attention_tree_hip, good, [
        {"q": f16(5, 200)}, {"q": f16(5, 256).float()}, {"q": f16(256, 5).t()}, {"q": f16(5, 0)}, {"q": f16(4, 256)}, {"kpages": f16(4, 1, 16, 128).float()}, {"vpages": f16(4, 1, 32, 128)},
        {"kpages": f16(2, 4, 1, 16, 128), "vpages": f16(2, 4, 1, 16, 128)}, {"kpages": f16(4, 1, 8, 128), "vpages": f16(4, 1, 8, 128)}, {"kpages": f16(4, 2, 16, 128), "vpages": f16(4, 2, 16, 128), "q": f16(5, 384)},
        {"block_table": i32(2, 4)}, {"block_table": i32(3, 4).long()}, {"block_table": i32(3, 0)}, {"block_table": i32(3, 8)[:, ::2]}, {"lengths": i32(2)}, {"granted": i64(3)}, {"starts": i32(5)}, {"masks": i32(5)},
        {"masks": i64(6)}, {"nodes": 0}, {"nodes": 65}, {"out": f16(5, 128)}, {"out": f16(5, 256).float()}, {"masks": torch.zeros(5, dtype=torch.int64)}])
    narrow = dict(good, q=f16(5, 192), kpages=f16(4, 1, 16, 96), vpages=f16(4, 1, 16, 96))
    with pytest.raises(RuntimeError, match="unsupported dimension"):
        IU.attention_tree_hip(**narrow)


def test_accept():
    good = dict(tokens=i64(5), parents=i32(5), targets=i64(5), slots=i64(5) - 1, lengths=i32(3), granted=i32(3), starts=i32(4), block_table=i32(3, 4), free_pages=i32(4), free_state=i32(2),
                kpages=f16(2, 4, 1, 16, 64), vpages=f16(2, 4, 1, 16, 64), nodes=8)
    refuse(IU.tree_accept_hip, good, [
        {"tokens": i32(5)}, {"tokens": i64(4)}, {"parents": i64(5)}, {"targets": i32(5)}, {"slots": i32(5)}, {"slots": i64(10)[::2]}, {"lengths": i32(4)}, {"starts": i32(3)}, {"block_table": i32(4, 4)},
        {"free_pages": i32(5)}, {"free_pages": i64(4)}, {"free_state": i32(3)}, {"kpages": f16(2, 4, 1, 16, 64).float()}, {"vpages": f16(1, 4, 1, 16, 64)}, {"kpages": f16(2, 4, 1, 16, 60), "vpages": f16(2, 4, 1, 16, 60)},
        {"kpages": f16(4, 1, 16), "vpages": f16(4, 1, 16)}, {"kpages": f16(2, 4, 1, 24, 64), "vpages": f16(2, 4, 1, 24, 64)}, {"nodes": 0}, {"nodes": 65}])


def test_fork():
    good = dict(source=i32(3), lengths=i32(3), block_table=i32(3, 4), free_pages=i32(4), free_state=i32(2), shares=i32(4), kpages=f16(2, 4, 1, 16, 64), vpages=f16(2, 4, 1, 16, 64))
    refuse(IU.page_fork_hip, good, [
        {"source": i64(3)}, {"source": i32(2)}, {"lengths": i32(4)}, {"block_table": i32(2, 4)}, {"block_table": i32(3, 0)}, {"free_pages": i32(5)}, {"free_state": i64(2)}, {"shares": i32(3)}, {"shares": i64(4)},
        {"kpages": f16(2, 4, 1, 16, 64).float()}, {"vpages": f16(2, 4, 1, 32, 64)}, {"kpages": f16(2, 4, 1, 16, 12), "vpages": f16(2, 4, 1, 16, 12)},
        {"kpages": f16(2, 4, 1, 16, 128)[..., ::2], "vpages": f16(2, 4, 1, 16, 128)[..., ::2]}])


def test_adjust():
    good = dict(logits=f16(4, 100), history=i32(3, 9), history_lengths=i32(3), prompt_lengths=i32(3), repetition=f32(3), frequency=f32(3), presence=f32(3), drafted=i32(4, 2), requests=i32(4),
                bias_tokens=i32(3, 5), bias=f32(3, 5), allowed=i32(2, 4), allowed_rows=i32(4), out=None)
    refuse(IU.logits_adjust_hip, good, [
        {"logits": f16(4, 100).float()}, {"logits": f16(400)}, {"logits": f16(100, 4).t()}, {"logits": f16(1, 100).expand(4, 100)}, {"logits": f16(5, 100)}, {"history": i64(3, 9)}, {"history": i32(2, 9)}, {"history": i32(27)},
        {"history": i32(3, 18)[:, ::2]}, {"history": None}, {"history_lengths": i32(4)}, {"prompt_lengths": i64(3)}, {"repetition": f16(3)}, {"frequency": f32(4)}, {"presence": f32(3, 1)}, {"drafted": i32(3, 2)}, {"drafted": i64(4, 2)},
        {"requests": i64(4)}, {"requests": i32(3)}, {"requests": None}, {"bias_tokens": i32(3, 4)}, {"bias_tokens": None}, {"bias": None}, {"bias": f16(3, 5)}, {"allowed": i32(2, 3)}, {"allowed": i32(2, 5)}, {"allowed": None},
        {"allowed": i64(2, 4)}, {"allowed_rows": None}, {"allowed_rows": i64(4)}, {"allowed_rows": i32(3)}, {"out": f16(4, 99)}, {"out": f16(4, 100).float()}, {"out": f16(100, 4).t()},
        {"history": None, "history_lengths": None, "prompt_lengths": None, "drafted": None}, {"allowed_rows": torch.zeros(4, dtype=torch.int32)}])
