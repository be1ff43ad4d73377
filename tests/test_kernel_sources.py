"""Rules of the hardware that no run can show to be kept, checked in the kernels' sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rllama_b200", "csrc")


@pytest.mark.parametrize("path", sorted(p for p in glob.glob(os.path.join(CSRC, "*.cu")) if "setmaxnreg" in open(p).read()), ids=os.path.basename)
def test_a_warpgroup_changes_its_registers_at_one_instruction(path):
    """setmaxnreg has to be the same instruction for all warps of a warpgroup: one place that gives registers away and one that takes them,
    for whole warpgroups, not one in each branch of the warps' roles."""
    code = re.sub(r"//[^\n]*", "", open(path).read())
    for what in ("dec", "inc"):
        assert code.count("setmaxnreg." + what) == 1
    assert re.search(r"static_assert\(MMA_WARP % 4 == 0 && THREADS % 128 == 0", code)
