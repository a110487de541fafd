"""Tree attention's loop over the stages has barriers of its own, which wait for nothing.  In the assembly every LDS write of a wave is waited for before the next barrier, so that the other waves' writes
to the same place come behind it."""
import os
import re
import subprocess

import pytest

from test_build_resources import CSRC, FLAGS, HIPCC

WRITE = re.compile(r"^\s+ds_(write|store|or|and|add|min|max|cmpst|wrxchg)")
WAIT = re.compile(r"^\s+s_waitcnt\b.*lgkmcnt\(0\)")


def writes_across_barriers(lines):
    """(write, barrier) line numbers, in the order of the text: what is between them waits for no LDS write."""
    found, pending = [], []
    for n, line in enumerate(lines):
        if WRITE.match(line):
            pending.append(n)
        elif WAIT.match(line):
            pending = []
        elif re.match(r"^\s+s_barrier", line):
            found += [(w, n) for w in pending]
            pending = []
    return found


def test_the_search_finds_one():
    text = "\tds_write_b32 v1, v2\n\ts_waitcnt vmcnt(0)\n\ts_barrier\n\tds_or_b32 v1, v2\n\ts_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier"
    assert writes_across_barriers(text.split("\n")) == [(0, 2)]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_lds_writes_are_waited_for(tmp_path):
    asm = tmp_path / "k.s"
    out = subprocess.run([HIPCC] + FLAGS + ["-w", "-S", "--cuda-device-only", os.path.join(CSRC, "tree_attention.hip"), "-o", str(asm)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-2000:]
    text, kernels = asm.read_text(), 0
    for name in re.findall(r"^(_ZN\S*attention_tree_\S*kernel\S*):", text, re.M):
        body = text[text.index(f"\n{name}:"):]
        lines = body[:body.index(".Lfunc_end")].split("\n")
        across = writes_across_barriers(lines)
        assert not across, (name, [(lines[w].strip(), b - w) for w, b in across])
        kernels += any("s_barrier" in line for line in lines)
    assert kernels >= 14                          # eight builds for few rows, six for more
