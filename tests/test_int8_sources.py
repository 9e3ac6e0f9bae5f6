"""What the sources of the 8-bit row kernels have to keep to and no run shows reliably."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "circuit-rag_b200", "csrc")


@pytest.mark.parametrize("name", ["int8.cuh", "int8_rows.h", "int8_rows.cuh", "int8_rows.cu", "int8_scores.cu"])
def test_no_non_coherent_loads(name):
    """These kernels start while the one before them on the stream still writes what they will read: the non-coherent
    path (which may be read ahead of the wait) is only for data that nobody writes during a kernel's life."""
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.search(r"__ldg\s*\(|ld\.global\.nc|__restrict__", code)
