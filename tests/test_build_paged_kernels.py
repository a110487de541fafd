"""The assembly checks of test_build_resources.py and test_build_more_kernels.py for the kernels of requests of unequal lengths: no scratch memory."""
import os
import re
import subprocess

import pytest

from test_build_resources import CSRC, FLAGS, HIPCC


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("src", ["paged.hip", "paged_attention.hip", "sample.hip"])
def test_no_scratch_memory(src, tmp_path):
    asm = tmp_path / "k.s"
    out = subprocess.run([HIPCC] + FLAGS + ["-w", "-S", "--cuda-device-only", os.path.join(CSRC, src), "-o", str(asm)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-2000:]
    text = asm.read_text()
    sizes = [int(v) for v in re.findall(r"\.private_segment_fixed_size:\s+(\d+)", text)]
    assert sizes and max(sizes) == 0 and not re.search(r"^\s+scratch_(load|store)", text, re.M)
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
