"""Kernels that are launched as programmatic dependents run before the kernel ahead of them has ended, and may not read what
that one writes through the read-only path: such a load is one of memory that nobody writes while the kernel runs, and the
compiler may move it ahead of the wait.  A layer's operands, its key mask, gain and scales among them, can all come from the
kernel ahead.  (The sources are searched: a stale value depends on the moment.)"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "brodiffusion_b200", "csrc")
READ_ONLY = re.compile(r"__ldg\s*\(|ld\.global\.nc|__restrict__")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return [line.split("//")[0] for line in f]


@pytest.mark.parametrize("name", ["add_rmsnorm.cu", "gemm_few.cu", "gemm_layer.cuh", "sdpa_window.cu", "sdpa_window.cuh"])
def test_a_layers_operands_are_not_read_through_the_read_only_path(name):
    assert [line for line in code(name) if READ_ONLY.search(line)] == []


def test_the_key_mask_of_the_tensor_core_kernel_is_not_either():
    assert [line for line in code("sdpa_tc05.cu") if READ_ONLY.search(line) and "key_mask" in line] == []
