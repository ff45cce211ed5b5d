"""Products with 4-bit weights at the sizes of a large model's layers, which reach every kernel of the operator with K over
one CTA and over clusters, row tiles in odd numbers and ragged ends of K, and at the ends of BF16's range.  Tolerances as in
test_linear_w4_gpu.py."""
import os
import subprocess
import sys

import pytest
import torch

from four_bit import randn
from test_linear_w4_gpu import check, pack, run, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k,ms", [(10230, 2560, (1, 8, 12, 16)), (5111, 5120, (1, 8, 32, 48)), (2551, 2568, (1, 7, 24)), (2551, 10240, (1, 8, 12, 16, 32, 48)),
                                    (5111, 5000, (5, 13)), (13810, 4104, (1, 8)), (20471, 1032, (1, 20)), (1291, 10240, (3, 40)), (4711, 1928, (8, 9)), (5111, 1288, (24,))])
def test_sizes_of_large_layers(bd, n, k, ms, group, dtype):
    codes, scales = weights(n + k, n, k, group, dtype)
    packed = pack(bd, codes, scales, group)
    for m in ms:
        x = randn(m, m, k, dtype=dtype)
        bias, gate, residual = randn(1, n, dtype=dtype), randn(2, n, dtype=dtype), randn(3, m, n, dtype=dtype)
        check(run(bd, x, packed, n, group, bias, act="silu", gate=gate, residual=residual), x, codes, scales, group, bias, gate, residual, "silu")


def exact_codes(n, k):
    return (torch.arange(n * k, device="cuda") * 7 % 16).view(n, k).double()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 11])
@pytest.mark.parametrize("size", [2.0 ** 58, 2.0 ** 60, 2.0 ** 62])
def test_sums_of_large_activations(bd, size, m, group):
    """Every value is within the range that counts, their sum over a group is far beyond it."""
    n, k = 40, 512
    codes = exact_codes(n, k)
    scales = torch.stack([randn(1, n, k // group), randn(2, n, k // group)], -1)
    x = (randn(3, m, k, dtype=torch.float32).abs().clamp(0.5, 1.9) * size).bfloat16()
    check(run(bd, x, pack(bd, codes, scales, group), n, group), x, codes, scales, group)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 11])
@pytest.mark.parametrize("size", [2.0 ** 57, 2.0 ** 62, 2.0 ** 100, 2.0 ** -100])
def test_steps_of_any_size(bd, size, m, group):
    """(and rows of X that are zero, which stay zero)"""
    n, k = 40, 512
    codes = exact_codes(n, k)
    scales = torch.stack([randn(1, n, k // group, dtype=torch.float32) * size, randn(2, n, k // group, dtype=torch.float32) * size], -1).bfloat16()
    x = randn(3, m, k)
    x[0, :256] = 0
    packed = pack(bd, codes, scales, group)
    check(run(bd, x, packed, n, group), x, codes, scales, group)
    assert (run(bd, torch.zeros_like(x), packed, n, group) == 0).all()


CAPTURED_FIRST = """
import torch, brodiffusion_b200 as bd
r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
xs = [r(m, 5120) for m in (1, 8, 16, 48)]
w = torch.empty(bd.w4_bytes(5111, 5120, 32), device="cuda", dtype=torch.uint8)
codes = torch.randint(0, 256, (5111, 2560), device="cuda", dtype=torch.uint8)
pairs = (0.1 * torch.randn(5111, 160, 2, device="cuda")).bfloat16()
ys = [torch.zeros(len(x), 5111, device="cuda", dtype=torch.bfloat16) for x in xs]
calls = lambda: (bd.w4_pack(codes, pairs, w, group=32), [bd.linear_w4_fwd(x, w, None, y, group=32) for x, y in zip(xs, ys)])
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls()
g.replay()
torch.cuda.synchronize()
first = [y.clone() for y in ys]
[y.zero_() for y in ys]
calls()
assert all(y.float().std() > 1 for y in first) and all(torch.equal(a, b) for a, b in zip(first, ys)) and bd.device_status() == 0
print("captured first")
"""


def test_a_processs_first_products_are_captured():
    res = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], capture_output=True, text=True, timeout=300,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert res.returncode == 0 and "captured first" in res.stdout, res.stderr[-2000:]
