"""Which kernel, tile width and split a layer's product gets (csrc/gemm_plan.h, compiled here)."""
import ctypes as C
import os
import random
import subprocess

import pytest

from layer_shapes import SHAPES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("plan") / "plan.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-o", so, os.path.join(ROOT, "tests", "cpp", "layer_plan_probe.cpp")])
    lib = C.CDLL(so)

    def run(M, N, K, act, sms=148):
        out = (C.c_int * 3)()
        lib.probe_layer_plan(M, N, K, int(act), sms, out)
        return "pair" if out[0] else "one", out[1], out[2]
    return run


@pytest.mark.parametrize("M,N,K,act,kernel,cols,split", SHAPES)
def test_the_shapes_take_the_kernels_they_are_for(plan, M, N, K, act, kernel, cols, split):
    assert plan(M, N, K, act) == (kernel, cols, split)


def test_every_plan_is_one_the_kernels_have(plan):
    rng = random.Random(1)
    for _ in range(20000):
        M, N, K = rng.randint(1, 5000), 8 * rng.randint(1, 1500), 8 * rng.randint(1, 1500)
        kernel, cols, split = plan(M, N, K, rng.random() < 0.5, rng.choice([2, 74, 132, 148, 160]))
        if kernel == "pair":
            assert cols in (128, 160, 192, 224, 256) and N % cols == 0 and split == 1
        else:
            assert cols in (32, 64, 80, 96, 112, 128) and split in (1, 2, 4, 8) and split <= (K + 63) // 64
            assert split == 1 or cols in (64, 96)
