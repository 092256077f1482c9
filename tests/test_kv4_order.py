"""What the 4-bit cache's early-starting kernels may read, from their source: no GPU."""
import os
import re

import ridgefill_data_b200

CSRC = os.path.join(os.path.dirname(ridgefill_data_b200.__file__), "csrc")


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_early_starting_kernels_take_no_read_only_loads():
    """A kernel that starts before its predecessor has ended runs while tables, positions and rows may still be written. Its
    wait orders ordinary loads alone: a load through the read-only path states that the data does not change while the kernel
    runs, and may be moved above the wait."""
    early = [n for n in sorted(os.listdir(CSRC)) if n.endswith(".cu") and "wait_previous()" in _code(n)]
    assert early == ["kv4_attention.cu"]
    for name in early:
        code = _code(name)
        assert not re.search(r"__ldg|ld\.global\.nc|__restrict__|kv4_block", code), name
        # in each kernel the wait comes before the first access through the arguments' pointers
        for body in re.findall(r"__global__.*?\n}\n", code, re.S):
            first = re.search(r"a\.(pos\[|c\.pages|q \+|part_|gate|out \+|c\.pool)", body)
            assert 0 <= body.find("wait_previous()") < first.start(), name
