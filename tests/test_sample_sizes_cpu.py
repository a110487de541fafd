"""bs_sample_f16 takes every size that its description allows: V up to 2^18, B up to 2^20, B * V up to 2^33."""
import pytest

from bitstack_amd import _lib


@pytest.mark.parametrize("V", [1, 511, 512, 513, 8191, 8192, 8193, 32700, 50257, 128256, 262143, 262144])
def test_largest_batches(V):
    L = _lib.lib()
    B = min(2 ** 20, 2 ** 33 // V)
    assert L.bs_sample_workspace_bytes(B, V) >= 16 * B * -(-V // 512)
    assert L.bs_sample_workspace_bytes(B + 1, V) == -2
