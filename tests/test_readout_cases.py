"""The read-out operators' sources, sizes and refusals that need no GPU."""
import glob
import os
import re

from pink_b200 import build


def test_waits_for_tensor_memory_name_the_registers_they_wait_for():
    """A wait that names no registers orders nothing for the compiler: uses of loaded values could move before it."""
    waits = 0
    for path in glob.glob(os.path.join(build.CSRC, "*.cu*")):
        text = open(path).read()
        for at in re.finditer(r"tcgen05\.wait::ld", text):
            waits += 1
            assert '"+r"(v[0])' in text[at.start():text.index(");", at.start())], path
    assert waits >= 2
