"""Kernels of the operators on device memory may run while the kernels before them still write (they are launched that way), so that none of them may read through the read-only path, which is defined only for
memory that nobody writes while the kernel is there: neither by the intrinsic nor by pointers that the compiler may take for constant."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "goneuron_b200", "csrc")
FILES = ["device_ops.cuh", "operators.cu"] + sorted(f for f in os.listdir(CSRC) if f.startswith("op_"))


@pytest.mark.parametrize("name", FILES)
def test_no_loads_of_the_read_only_path(name):
    text = re.sub(r"//.*", "", open(os.path.join(CSRC, name)).read())
    assert not re.findall(r"\b__ldg\b|\b__restrict__\b|\bld\.global\.nc\b", text)
