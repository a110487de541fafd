"""What the Python entry points for requests of unequal lengths refuse: types, shapes and layouts that the kernels do not take, before anything is launched."""
import pytest
import torch

from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32, device="cuda")


def f16(*shape):
    return torch.zeros(*shape, dtype=torch.float16, device="cuda")


def refuse(fn, good, cases):
    fn(**good)
    for change in cases:
        with pytest.raises((ValueError, RuntimeError)):
            fn(**{**good, **change})


def test_plan():
    good = dict(lengths=i32(3), new_tokens=i32(3), block_table=i32(3, 4), free_pages=i32(9), free_state=i32(2), page_size=16, tokens=3, released=None)
    refuse(IU.page_plan_hip, good, [
        {"lengths": i32(3).long()}, {"lengths": i32(4)}, {"lengths": i32(3, 1)}, {"new_tokens": i32(2)}, {"new_tokens": i32(6)[::2]}, {"block_table": i32(4, 3)}, {"block_table": i32(3, 8)[:, :4]},
        {"block_table": i32(3, 4).long()}, {"block_table": i32(3, 0)}, {"free_pages": i32(9).long()}, {"free_pages": i32(3, 3)}, {"free_pages": i32(0)}, {"free_state": i32(3)}, {"page_size": 8}, {"page_size": 20}, {"tokens": -1},
        {"released": i32(3)}, {"released": i32(2).bool()}, {"released": torch.zeros(3, dtype=torch.bool)}])


def test_store():
    good = dict(q=f16(5, 256), k=f16(5, 128), v=f16(5, 128), cos=f16(9, 64), sin=f16(9, 64), kpages=f16(4, 1, 16, 128), vpages=f16(4, 1, 16, 128), positions=i32(5),
                slots=torch.arange(5, device="cuda"), out=None)
    refuse(IU.rope_store_paged_hip, good, [
        {"q": f16(5, 200)}, {"q": f16(4, 256)}, {"q": f16(5, 256).float()}, {"q": f16(256, 5).t()}, {"q": f16(5, 0)}, {"k": f16(5, 256)}, {"k": f16(4, 128)}, {"v": f16(5, 256)[:, :128]}, {"v": f16(5, 128).float()},
        {"cos": f16(9, 32)}, {"cos": f16(8, 64)}, {"cos": f16(9, 64).float()}, {"kpages": f16(4, 1, 16, 64)}, {"kpages": f16(4, 16, 1, 128).transpose(1, 2)[:, :, ::2]}, {"vpages": f16(3, 1, 16, 128)},
        {"kpages": f16(4, 1, 8, 128), "vpages": f16(4, 1, 8, 128)}, {"positions": i32(5).long()}, {"positions": i32(6)}, {"slots": i32(5)}, {"out": f16(5, 128)}, {"out": f16(5, 256).float()},
        {"q": None, "out": f16(5, 256)}, {"q": torch.zeros(5, 256).half()}])
    narrow = dict(good, q=f16(5, 192), k=f16(5, 96), v=f16(5, 96), cos=f16(9, 48), sin=f16(9, 48), kpages=f16(4, 1, 16, 96), vpages=f16(4, 1, 16, 96))
    with pytest.raises(RuntimeError, match="unsupported dimension"):
        IU.rope_store_paged_hip(**narrow)


def test_attention():
    good = dict(qkv=f16(3, 512), kpages=f16(4, 1, 16, 128), vpages=f16(4, 1, 16, 128), cos=f16(99, 64), sin=f16(99, 64), block_table=i32(3, 4), lengths=i32(3),
                slots=torch.full((3,), -1, device="cuda"), heads=2, kv_heads=1, out=None)
    refuse(IU.attention_paged_hip, good, [
        {"qkv": f16(3, 384)}, {"qkv": f16(2, 512)}, {"qkv": f16(3, 512).float()}, {"qkv": f16(512, 3).t()}, {"kv_heads": 2}, {"heads": 3}, {"heads": 0}, {"block_table": i32(2, 4)},
        {"block_table": i32(3, 4).long()}, {"block_table": i32(3, 0)}, {"lengths": i32(2)}, {"lengths": i32(3).long()}, {"slots": i32(3)}, {"slots": torch.zeros(4, dtype=torch.int64, device="cuda")},
        {"cos": f16(0, 64), "sin": f16(0, 64)}, {"sin": f16(98, 64)}, {"vpages": f16(4, 1, 32, 128)}, {"kpages": f16(4, 1, 16, 128).float()}, {"out": f16(3, 128)}, {"out": f16(3, 256).float()},
        {"lengths": torch.zeros(3, dtype=torch.int32)}])


def test_sample():
    good = dict(logits=f16(3, 100), uniform=torch.zeros(3, device="cuda"), temperature=None, top_k=None, top_p=None, min_p=None, out=None)
    numbers = torch.zeros(3, device="cuda")
    refuse(IU.sample_hip, good, [
        {"logits": f16(3, 100).float()}, {"logits": f16(300)}, {"logits": f16(100, 3).t()}, {"logits": f16(4, 100)}, {"logits": f16(3, 0)}, {"logits": f16(1, 100).expand(3, 100)}, {"logits": f16(3, 2 ** 18 + 1)},
        {"uniform": numbers.double()}, {"uniform": numbers[:2]}, {"uniform": None}, {"temperature": numbers.half()}, {"top_k": numbers}, {"top_k": numbers.long()}, {"top_p": numbers[:, None]},
        {"min_p": torch.zeros(6, device="cuda")[::2]}, {"out": i32(3)}, {"out": torch.zeros(2, dtype=torch.int64, device="cuda")}, {"uniform": torch.zeros(3)}])
