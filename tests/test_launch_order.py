"""Programmatic dependent launch, read from the kernels' sources: dependents are signalled after the kernel's own wait."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fastgate_b200", "csrc")


def test_dependents_are_signalled_after_the_wait():
    """A linear reads its weight before its wait.  A kernel B that signals before its own wait lets the linear behind it start while
    the kernel in front of B still writes; signalled in the statement after the wait, it cannot."""
    found = 0
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".cu", ".cuh")) or name == "fg_ptx.cuh":
            continue
        with open(os.path.join(CSRC, name)) as f:
            code = [re.sub(r"//.*", "", line).strip() for line in f]
        code = [line for line in code if line]
        for i, line in enumerate(code):
            if "griddep_launch_dependents" in line:
                found += 1
                assert line == "griddep_launch_dependents();" and code[i - 1] == "griddep_wait();", (name, code[i - 1: i + 1])
    assert found >= 10
