"""Rules of the head's kernels that no run can show to be kept (CPU): their sources are read."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "noetic_tensor_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_shared_arrays_are_read_as_what_they_are_aligned_for():
    """No array of single bytes in shared memory is read in words: only its type aligns an array."""
    text = source("head_ops.cuh")
    assert not re.findall(r"__shared__\s+u?int8_t", text)
