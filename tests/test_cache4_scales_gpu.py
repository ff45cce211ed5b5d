"""Attention over the 4-bit cache where the steps of V are beyond what FP16 holds, or not finite."""
import math

import pytest
import torch

from four_bit import UNIT, held, quantised, randn, values
from test_cache4_gpu import garbage, run

pytestmark = pytest.mark.gpu


def attend(bd, q, k, v, heads, kv_heads, group, **kw):
    cache = garbage(bd, k.shape[0], kv_heads, k.shape[1], k.shape[2] // kv_heads, group, k.dtype)
    bd.cache4_append(k, v, cache)
    return run(bd, q, cache, heads, **kw)


@pytest.mark.parametrize("hd,group", [(64, 64), (64, 32), (128, 32), (128, 128)])
@pytest.mark.parametrize("lq", [1, 9])
@pytest.mark.parametrize("size,mix", [(2.0 ** -108, 0), (2.0 ** -112, 0), (2.0 ** -114, 0), (2.0 ** -115, 5)])
def test_tiny_values(bd, size, mix, lq, hd, group):
    """Steps of V from 2^-110 to 2^-118, alike or other by up to 2^mix from key to key."""
    n = 100
    q, k, v = randn(1, 1, lq, 2 * hd), randn(2, 1, n, hd), randn(3, 1, n, hd, dtype=torch.float32)
    v = (v * size * 2.0 ** (torch.arange(n, device="cuda") % (mix + 1))[:, None]).bfloat16()
    out = attend(bd, q, k, v, 2, 1, group)
    kd, (vc, vs) = held(k, group)[0], quantised(v[0], group)
    vd, step = values(vc, vs, group), vs.double().repeat_interleave(group, -2)[..., 0]
    seen = torch.arange(n, device="cuda")[None] <= n - lq + torch.arange(lq, device="cuda")[:, None]
    for h in range(2):
        s = (q[0, :, h * hd:(h + 1) * hd].double() @ kd.T / math.sqrt(hd)).masked_fill(~seen, -math.inf)
        p = torch.softmax(s, 1)
        ref = p @ vd
        # a weight's rounding to FP16, the scores' (4 * 2^-20 of 100 or less) and the sums' as in test_cache4_gpu.py; what is below FP32's
        # normal range counts as 0, once in a product of a weight and a value (a key) and once in a sum
        tol = UNIT[q.dtype] * ref.abs() + (2.0 ** -11 + 2.0 ** -17) * (p @ (step * (vc - 8).abs())) + 2.0 ** -11 * (p @ ((vd - 8 * step).abs() + 8 * step)) + 3 * n * 2.0 ** -126
        err = (out[0, :, h * hd:(h + 1) * hd].double() - ref).abs()
        assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("at", [3, 20, 58])
@pytest.mark.parametrize("lq", [1, 5])
def test_a_visible_row_that_is_not_finite_reaches_the_output_whatever_its_weight(bd, at, lq):
    """0 times NaN is NaN, whether or not all queries see all of the sixteen keys that the row lies among."""
    hd, n = 64, 60
    q = randn(1, 1, lq, hd).abs() + 1
    k, v = randn(2, 1, n, hd), randn(3, 1, n, hd)
    k[0, at], v[0, at, :32] = -1000.0, float("nan")          # a score of -8000 and less
    out = attend(bd, q, k, v, 1, 1, 32)
    for i in range(lq):
        sees = n - lq + i >= at
        assert torch.isnan(out[0, i, :32]).all() == sees and torch.isfinite(out[0, i, 32:]).all(), (i, sees)
    mask = torch.ones(n, device="cuda")
    mask[at] = 0
    assert torch.isfinite(attend(bd, q, k, v, 1, 1, 32, key_mask=mask)).all()
