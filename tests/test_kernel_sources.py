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


def loads_of_tensor_memory(text):
    """The line before each load (or run of loads) of tensor memory."""
    lines = [line.strip() for line in text.splitlines() if line.strip()]
    is_load = [line.startswith(("tc_ld32(", "tc_ld16(")) for line in lines]
    return [lines[i - 1] for i in range(1, len(lines)) if is_load[i] and not is_load[i - 1]]


def test_a_warp_comes_together_before_it_loads_tensor_memory():
    """tcgen05.ld is executed by a whole warp (.sync.aligned), and the code before it in a loop is not the same in every lane."""
    before = loads_of_tensor_memory(source("head_gemm.cuh"))
    assert len(before) == 4 and set(before) == {"__syncwarp();"}
    assert loads_of_tensor_memory(source("readout.cuh")) == ["__syncwarp();"]


def test_a_warp_gives_up_a_wait_as_one():
    """Behind a wait for an accumulator the warp's lanes meet again: one that gave up by itself would leave the others waiting for it."""
    for name, waits in (("head_gemm.cuh", 1), ("readout.cuh", 2)):
        lines = [line for line in source(name).splitlines() if "mbar_wait(bar_acc_full" in line]
        assert len(lines) == waits and all("__all_sync(0xffffffffu, mbar_wait(" in line for line in lines)


def test_what_crosses_between_the_ctas_of_a_pair_says_so():
    """Arrivals on the other CTA's barrier, and the waits for them, are ordered for the cluster: the default is the own CTA."""
    for name in ("tcgen05.cuh", "head_gemm.cuh", "readout.cuh"):
        for arrival in re.findall(r"mbarrier\.arrive[\w.:]*", source(name)):
            assert "shared::cluster" not in arrival or re.search(r"\.(relaxed|release)\.cluster\.", arrival), arrival
    assert re.search(r"mbarrier\.try_wait\.parity\.\w+\.cluster\.", source("tcgen05.cuh"))
    assert re.findall(r"mbar_wait(<\w+>)?\(bar_acc_empty", source("head_gemm.cuh")) == ["<PAIR>"]
    assert re.findall(r"mbar_wait(<\w+>)?\(bar_acc_empty", source("readout.cuh")) == ["", "<true>"]  # one CTA, a pair


def test_kernels_that_start_early_read_nothing_as_read_only_data():
    """Such a kernel is running before the one that writes its inputs has ended, so they change during its lifetime."""
    for name in ("head_gemm.cuh", "head_ops.cuh"):
        assert not re.findall(r"__ldg\(|ldg_stream\w*\(|ld\.global\.nc|__restrict__", source(name)), name
