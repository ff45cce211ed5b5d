"""Attention over the 4-bit cache where the steps of V differ by more than FP16 holds: tiny ones, large ones in keys that a
query does not see, or that count for next to nothing, or in another group of the same row; and rows that are not finite.  Tolerances as
in test_cache4_gpu.py: they are of what a query sees, and of each column by itself."""
import math

import pytest
import torch

from four_bit import UNIT, held, quantised, randn, values
from test_cache4_gpu import check, garbage, run

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


LARGE = [(torch.bfloat16, 1e15), (torch.bfloat16, 1e30), (torch.float16, 3e4)]
SMALL = {torch.bfloat16: 1.0, torch.float16: 1e-3}


@pytest.mark.parametrize("dtype,large", LARGE)
@pytest.mark.parametrize("hd,group", [(64, 64), (64, 32), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("lq,heads", [(2, 1), (3, 2), (8, 1), (12, 2), (40, 2)])
def test_large_values_in_rows_that_come_later(bd, lq, heads, hd, group, dtype, large):
    """The drafted rows' V are far larger from row to row: the queries ahead of a row know nothing of it."""
    n = 70
    q, k, v = randn(1, 1, lq, heads * hd, dtype=dtype), randn(2, 1, n, hd, dtype=dtype), randn(3, 1, n, hd, dtype=dtype, scale=SMALL[dtype])
    v[0, -1] = randn(4, hd, dtype=torch.float32, scale=large / 4).clamp(-large, large).to(dtype)
    if lq > 2:
        v[0, -2] = randn(5, hd, dtype=torch.float32, scale=math.sqrt(large * SMALL[dtype])).to(dtype)
    check(attend(bd, q, k, v, heads, 1, group), q, k, v, heads, 1, group)


@pytest.mark.parametrize("dtype,large", LARGE)
@pytest.mark.parametrize("hd,group", [(64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("at", [0, 5, 40, 331])
@pytest.mark.parametrize("window,depth", [(0, 10.0), (0, 20.0), (100, 60.0)])
def test_large_values_of_keys_that_count_for_little(bd, window, depth, at, hd, group, dtype, large):
    """A key of large V whose weight is some e^-18, e^-36, e^-108: early, late, behind the window of most queries, hidden by the
    key mask of all."""
    n, lq = 333, 20
    # (queries of one sign, 1.8 on average, against a key of the other one)
    q = randn(1, 1, lq, hd, dtype=dtype).abs() + 1
    k, v = randn(2, 1, n, hd, dtype=dtype), randn(3, 1, n, hd, dtype=dtype, scale=SMALL[dtype])
    k[0, at] = -depth / math.sqrt(hd)
    v[0, at] = randn(4, hd, dtype=torch.float32, scale=large / 4).clamp(-large, large).to(dtype)
    check(attend(bd, q, k, v, 1, 1, group, window=window, sinks=3), q, k, v, 1, 1, group, window, 3)
    mask = torch.ones(n, device="cuda")
    mask[at] = 0
    check(attend(bd, q, k, v, 1, 1, group, window=window, key_mask=mask), q, k, v, 1, 1, group, window, 0, mask=mask)


@pytest.mark.parametrize("dtype,large", LARGE)
@pytest.mark.parametrize("lq,n", [(1, 40), (1, 3000), (30, 300)])
def test_the_largest_score_wins_over_an_earlier_large_value(bd, lq, n, dtype, large):
    """Keys of large V ahead of the one that takes nearly all: what is kept of the first ones fades with their weights."""
    hd, group = 128, 32
    q = randn(1, 1, lq, hd, dtype=dtype).abs() + 1
    k, v = randn(2, 1, n, hd, dtype=dtype), randn(3, 1, n, hd, dtype=dtype, scale=SMALL[dtype])
    v[0, 0:n // 3:7] = randn(4, len(range(0, n // 3, 7)), hd, dtype=torch.float32, scale=large / 4).clamp(-large, large).to(dtype)
    k[0, n // 2] = 60.0 / math.sqrt(hd)
    check(attend(bd, q, k, v, 1, 1, group), q, k, v, 1, 1, group)


@pytest.mark.parametrize("dtype,large", LARGE)
@pytest.mark.parametrize("hd,group", [(64, 32), (128, 32), (128, 64)])
@pytest.mark.parametrize("lq", [1, 4, 20])
def test_large_values_in_another_group_of_the_row(bd, lq, hd, group, dtype, large):
    """Each group of columns has the sum of its own values, as with values that are not finite."""
    n = 200
    q, k, v = randn(1, 1, lq, 2 * hd, dtype=dtype), randn(2, 1, n, hd, dtype=dtype), randn(3, 1, n, hd, dtype=dtype, scale=SMALL[dtype])
    v[0, ::3, :group] = randn(4, len(range(0, n, 3)), group, dtype=torch.float32, scale=large / 4).clamp(-large, large).to(dtype)
    v[0, :, -group:] *= 2.0 ** -6
    check(attend(bd, q, k, v, 2, 1, group), q, k, v, 2, 1, group)


@pytest.mark.parametrize("hd,group", [(64, 32), (128, 32), (128, 64)])
@pytest.mark.parametrize("lq,n", [(1, 600), (3, 3000), (20, 400)])
@pytest.mark.parametrize("late", [0.0, 1e-30, 1e-3, 1.0])
def test_groups_of_zeros(bd, late, lq, n, hd, group):
    """The columns of a narrower head, filled up with zeros; and ones that are no longer zero in the last third of the rows."""
    q, k, v = randn(1, 1, lq, 2 * hd), randn(2, 1, n, hd), randn(3, 1, n, hd)
    v[0, :, -group:] = 0
    v[0, n - n // 3:, -group:] = randn(4, n // 3, group, dtype=torch.float32, scale=late).bfloat16()
    out = attend(bd, q, k, v, 2, 1, group)
    check(out, q, k, v, 2, 1, group)
    if late == 0:
        assert (out.view(lq, 2, hd)[..., -group:] == 0).all()


@pytest.mark.parametrize("hd,group", [(64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("lq,window", [(1, 0), (8, 0), (33, 500)])
def test_rows_and_groups_of_every_size(bd, lq, window, hd, group):
    """Every group of every row by itself between 2^-60 and 2^60 times the usual size, scores spread over some hundred."""
    n = 2000
    q, k, v = randn(1, 1, lq, 2 * hd, scale=6.0), randn(2, 1, n, hd), randn(3, 1, n, hd, dtype=torch.float32)
    sizes = torch.randint(-60, 61, (1, n, hd // group), device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    v = (v * (2.0 ** sizes.double()).float().repeat_interleave(group, -1)).bfloat16()
    check(attend(bd, q, k, v, 2, 1, group, window=window, sinks=5), q, k, v, 2, 1, group, window, 5)


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
