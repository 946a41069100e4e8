"""The tracked head of the C++ host mirror under masks, temperatures and sums of terms: its test program passes on the GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = os.path.join(ROOT, "tests", "cpp", "test_head_tape.cpp")
PROGRAM = os.path.join(ROOT, "tests", "cpp", "_build", "test_head_tape")


def _program():
    from noetic_tensor_b200 import _build

    return _build.build_host_program(SOURCE, PROGRAM)


def test_program_compiles():
    import torch

    exe = _program()
    if not torch.cuda.is_available():
        r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
        assert r.returncode == 2 and "no CUDA device" in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
def test_program_passes():
    r = subprocess.run([_program()], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout[-3000:] + r.stderr[-2000:]
