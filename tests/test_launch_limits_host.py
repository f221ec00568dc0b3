"""How launchers ask for shared memory, read from their source (no GPU)."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quipsharp_b200", "csrc")
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


@pytest.mark.parametrize("name", SOURCES)
def test_no_limit_is_set_once_for_all_devices(name):
    """A kernel's limit belongs to a device; a function's static would set it on the first
    device that calls, and keep a failure for good."""
    text = open(os.path.join(CSRC, name)).read()
    assert not re.search(r"static\s[^;{}]*=\s*cudaFuncSetAttribute", text)
