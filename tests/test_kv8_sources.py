"""CPU: rules of the 8-bit K/V cache's CUDA sources that no run shows reliably."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "animaxs_b200", "csrc")


def test_early_launched_kernels_read_by_ordinary_loads():
    """A kernel that is resident while its predecessor still writes (pdl_wait) uses no non-coherent load: those are
    defined only for data that nobody writes during the kernel's whole life."""
    checked = 0
    for name in sorted(os.listdir(CSRC)):
        if not name.startswith("kv8_"):
            continue
        text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        checked += "pdl_wait()" in text
        assert not re.search(r"__ldg\s*\(|ld\.global\.nc|ld\.global\.L\w*::\w+\.nc", text), name
    assert checked >= 3
