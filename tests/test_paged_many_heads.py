"""attention_paged_hip with more KV heads than there are places for parts: nothing is cut, so that the first parts alone make the grid, whose 2^32 threads hold the
2^22 of them that the header allows, but not twice as many."""
import pytest
import torch

from bitstack_amd import _lib


def test_nothing_is_cut():
    bytes_of = _lib.lib().bs_attention_paged_workspace_bytes
    assert bytes_of(1, 768, 768, 64, 16, 4096) > 0
    for B, heads in ((1, 769), (1, 5000), (5, 4000), (1, 2 ** 22), (2, 2 ** 21), (64, 2 ** 16)):
        assert bytes_of(B, heads, heads, 64, 16, 4096) == 0, (B, heads)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv", [(768, 768), (769, 769), (1700, 850)])
def test_many_heads(heads, kv):
    from test_gpu_paged_attention import check
    check(heads, kv, 64, 16, [1100, 5, 0, 200])
