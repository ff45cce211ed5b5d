"""The norms around a block at the widest rows that a CTA's registers hold, on and off 16 bytes.  Tolerances as in
test_sandwich_norm_gpu.py."""
import pytest
import torch

from four_bit import randn
from test_sandwich_norm_gpu import E4M3, call, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 3, 200])
@pytest.mark.parametrize("cols", [16376, 16383, 16384, 16392])
def test_the_widest_rows(bd, cols, rows, dtype):
    x, r = randn(rows, rows, cols, dtype=dtype), randn(rows + 1, rows, cols, dtype=dtype)
    post, gain, gate = (1 + randn(cols + i, cols, dtype=dtype, scale=0.02) for i in range(3))
    for out in (None, dtype, E4M3):
        g = gain if out is not None else None
        check(call(bd, x, r, post, gate, 0.7, g, out), x, r, post, gate, 0.7, g)


@pytest.mark.parametrize("cols", [16370, 16376, 16384])
def test_the_widest_rows_off_sixteen_bytes(bd, cols):
    wide = randn(1, 2, 9, cols + 24)
    x, r = wide[0, :, 3:3 + cols], wide[1, :, 3:3 + cols]
    h, out = (torch.full_like(wide[0], 7.0)[:, 3:3 + cols] for _ in range(2))
    bd.sandwich_norm_fwd(x, r, h, out=out)
    check((h, out, None), x, r)
