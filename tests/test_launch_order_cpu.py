"""Kernels that start before the launch in front of them has ended: what their sources may do in which order.

A block that holds TMEM while it waits for another launch, or lets the next launch start while it has yet to take TMEM, can
lock the device up, and only where timing allows it: that order is read, not run."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "flydsl_b200" / "csrc"
WAIT, SIGNAL, BOTH = "wait_for_previous_launch()", "let_next_launch_start()", "after_previous_launch()"


def kernels():
    """(name, body) of every kernel in files that launch closely."""
    for path in sorted(CSRC.glob("*.cu")):
        text = path.read_text()
        if "launch_closely(" not in text:
            continue
        for m in re.finditer(r"^__global__.*?^}\n", text, re.S | re.M):
            name = re.search(r"(\w+)\(const", m.group(0)[m.group(0).index("__launch_bounds__"):].split(")", 1)[1])
            yield pytest.param(re.sub(r"//.*", "", m.group(0)), id=name.group(1))


def test_the_kernels_are_found():
    names = {p.id for p in kernels()}
    assert {"lora_shrink_kernel", "lora_fold_kernel", "lora_expand_kernel", "lora_wgrad_kernel", "lora_wgrad_finish_kernel",
            "lora_transpose_kernel", "lora_shrink_tc_kernel", "lora_expand_tc_kernel", "lora_wgrad_tc_kernel"} == names


@pytest.mark.parametrize("body", list(kernels()))
def test_tmem_is_taken_between_the_wait_and_the_signal(body):
    taken = [m.start() for m in re.finditer(r"tcgen05\.alloc", body)]
    if not taken:
        assert body.count(BOTH) == 1 and WAIT not in body and SIGNAL not in body
        return
    assert BOTH not in body and body.count(SIGNAL) == 1
    signal = body.index(SIGNAL)
    for at in taken:
        # the wait is the first thing in the branch of the warp that allocates, the signal comes after the whole block has met
        branch = body[:at].rindex("if (warp == ")
        assert WAIT in body[branch:at] and body[branch:at].index(WAIT) < 80
        assert "__syncthreads();" in body[at:signal]
    # everyone else waits as well before the first access to global memory
    met = body.index("__syncthreads();", taken[-1])
    assert body[met:signal].count(WAIT) == 1


@pytest.mark.parametrize("name", sorted(p.name for p in CSRC.glob("lora*")))
def test_nothing_is_read_through_the_read_only_path(name):
    """Their inputs may have been written by a launch that was still running when they started."""
    text = re.sub(r"//.*", "", (CSRC / name).read_text())
    assert not re.findall(r"__ldg|__restrict__|ld\.global\.nc", text)
    assert "vec8.cuh" not in text                # its loads are read-only ones
