"""rope_store_paged_hip against the rotation in 64 bits: what is copied is equal, what is rotated is off by the products' roundings in fp32 and one to fp16."""
import pytest
import torch

import paged_oracle as oracle
from bitstack_amd.utils import inference_utils as IU

pytestmark = pytest.mark.gpu


def tables(positions, d):
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return angles.cos().half().cuda(), angles.sin().half().cuda()


def near(got, x, cos, sin):
    """Each product and the sum are rounded in fp32 (2^-24 of each), the result to fp16 (2^-11, or half of the smallest step 2^-24)."""
    want = oracle.rotate(x, cos, sin)
    size = oracle.rotate(x.abs(), cos.abs(), -sin.abs())
    size = torch.maximum(size.abs(), oracle.rotate(x.abs(), cos.abs(), sin.abs()).abs())
    assert bool(((got.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -22 * size + 2.0 ** -25 * 1.01).all())


# tokens, heads, KV heads, head size, page, row padding of q and of k, v (0 and 8: 16 bytes at a time; others one value at a time)
SIZES = [(1, 1, 1, 64, 16, 0, 0), (1, 32, 8, 128, 16, 0, 0), (37, 4, 4, 128, 32, 8, 0), (300, 5, 1, 64, 1024, 0, 8), (129, 7, 7, 128, 64, 3, 1), (77, 16, 2, 64, 256, 8, 5)]


@pytest.mark.parametrize("T,heads,kv,d,page,padq,padkv", SIZES)
@pytest.mark.parametrize("how", ["inplace", "out", "keys"])
def test_store(T, heads, kv, d, page, padq, padkv, how):
    print(f"paged store T={T} heads={heads}/{kv} d={d} page={page} pads={padq},{padkv} {how}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T + d)
    pool, max_pos = T // page + 3, T + 50
    wide = torch.randn(T, heads * d + padq, device="cuda", generator=g).half()
    kv_wide = torch.randn(2, T, kv * d + padkv, device="cuda", generator=g).half()
    q, k, v = wide[:, :heads * d], kv_wide[0, :, :kv * d], kv_wide[1, :, :kv * d]
    cos, sin = tables(max_pos, d)
    kpages, vpages = torch.randn(2, pool, kv, page, d, device="cuda", generator=g).half()
    slots = torch.randperm(pool * page, device="cuda", generator=g)[:T]
    positions = torch.randint(0, max_pos, (T,), device="cuda", generator=g).int()
    # rows that are not stored: no slot, a slot or a position that does not exist
    if T > 10:
        slots[3], slots[5], slots[T - 1] = -1, pool * page, 2 ** 40
        positions[7], positions[8] = -1, max_pos
    live = (slots >= 0) & (slots < pool * page) & (positions >= 0) & (positions < max_pos)
    before = [t.clone() for t in (wide, kv_wide, kpages, vpages)]
    out = torch.full((T, heads * d + 2 * padq), 7.0, device="cuda", dtype=torch.float16)
    if how == "inplace":
        got = IU.rope_store_paged_hip(q, k, v, cos, sin, kpages, vpages, positions, slots)
        assert got is q and torch.equal(wide[:, heads * d:], before[0][:, heads * d:])
    elif how == "out":
        got = IU.rope_store_paged_hip(q, k, v, cos, sin, kpages, vpages, positions, slots, out=out[:, :heads * d])
        assert torch.equal(wide, before[0]) and bool((out[:, heads * d:] == 7.0).all())
    else:
        assert IU.rope_store_paged_hip(None, k, v, cos, sin, kpages, vpages, positions, slots) is None
        assert torch.equal(wide, before[0])
    at = positions.long().clamp(0, max_pos - 1)
    c, s = cos[at][:, None], sin[at][:, None]
    if how != "keys":
        old = before[0][:, :heads * d].unflatten(1, (heads, d))
        near(got.unflatten(1, (heads, d))[live], old[live], c[live], s[live])
        assert torch.equal(got.unflatten(1, (heads, d))[~live], old[~live])
    assert torch.equal(kv_wide, before[1])
    where, off = slots[live] // page, slots[live] % page
    near(kpages[where, :, off], k.unflatten(1, (kv, d))[live], c[live], s[live])
    assert torch.equal(vpages[where, :, off], v.unflatten(1, (kv, d))[live])
    rest = torch.ones(pool, page, dtype=torch.bool, device="cuda")
    rest[where, off] = False
    for pages, old in ((kpages, before[2]), (vpages, before[3])):
        assert torch.equal(pages.transpose(1, 2)[rest], old.transpose(1, 2)[rest])


def test_as_the_prompt_kernel_does_it():
    """The same values as rope_store_hip leaves in a cache without pages, bit for bit."""
    B, n, heads, kv, d, page = 2, 45, 8, 2, 128, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(B * n, h * d, device="cuda", generator=g).half() for h in (heads, kv, kv))
    cos, sin = tables(64, d)
    kcache, vcache = torch.zeros(2, B, kv, 64, d, device="cuda", dtype=torch.float16)
    q1, q2 = q.clone(), q.clone()
    IU.rope_store_hip(q1, k, v, cos, sin, kcache, vcache, n)
    kpages, vpages = torch.zeros(2, B * 4, kv, page, d, device="cuda", dtype=torch.float16)
    positions = torch.arange(n, device="cuda", dtype=torch.int32).repeat(B)
    slots = positions.long() + 64 * torch.arange(B, device="cuda").repeat_interleave(n)
    IU.rope_store_paged_hip(q2, k, v, cos, sin, kpages, vpages, positions, slots)
    assert torch.equal(q1, q2)
    for pages, cache in ((kpages, kcache), (vpages, vcache)):
        assert torch.equal(pages.view(B, 4, kv, page, d).transpose(1, 2).reshape(B, kv, 64, d), cache)


def test_pool_beyond_32_bits_of_values():
    """The last page of a pool of 2.3e9 values."""
    kv, page, d = 1, 1024, 128
    pool = 2 ** 31 // (page * d) + 1200
    kpages = torch.zeros(pool, kv, page, d, device="cuda", dtype=torch.float16)
    vpages = torch.zeros_like(kpages)
    k, v = torch.randn(2, 2, kv * d, device="cuda").half()
    cos, sin = torch.ones(4, d // 2, device="cuda").half(), torch.zeros(4, d // 2, device="cuda").half()
    slots = torch.tensor([pool * page - 1, 5], device="cuda")
    IU.rope_store_paged_hip(None, k, v, cos, sin, kpages, vpages, torch.tensor([1, 2], dtype=torch.int32, device="cuda"), slots)
    assert torch.equal(kpages[-1, 0, -1], k[0]) and torch.equal(vpages[-1, 0, -1], v[0]) and torch.equal(kpages[0, 0, 5], k[1])
    assert int(torch.count_nonzero(kpages[pool - 1])) <= d and int(torch.count_nonzero(kpages[1:pool - 1:97])) == 0
