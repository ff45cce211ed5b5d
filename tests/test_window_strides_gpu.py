"""Windowed attention of tensors with one row or one batch item, whose stride says nothing."""
import pytest
import torch

import test_sdpa_window_gpu as W

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 160])
@pytest.mark.parametrize("row,item", [(1, 1), (0, 0), (3, 5), (8, 12), (10 ** 6 + 1, 7)])
def test_strides_of_a_single_row_and_item_may_be_anything(bd, hd, row, item):
    nh = 4
    q, k, v = W.inputs(hd, 1, 1, 1, nh, nh, hd)
    odd = lambda t: t.as_strided((1, 1, nh * hd), (item, row, 1))
    out = torch.full_like(q, float("nan"))
    bd.sdpa_window_fwd(odd(q), odd(k), odd(v), odd(out), nh, window=3)
    assert bd.device_status() == 0 and torch.equal(out, v)             # one key: its value
    flat = torch.full_like(q[0], float("nan"))
    bd.sdpa_window_fwd(q[0].t().contiguous().t(), k[0].t().contiguous().t(), v[0], flat, nh, window=3)
    assert torch.equal(flat, v[0])
    q, k, v = W.inputs(hd + 1, 1, 5, 70, nh, nh, hd)                   # several rows of one item
    odd = lambda t: t.as_strided(t.shape, (item, nh * hd, 1))
    out = torch.full_like(q, float("nan"))
    bd.sdpa_window_fwd(odd(q), odd(k), odd(v), odd(out), nh, window=30)
    W.check(bd, q, k, v, nh, nh, 30, 0, out=out)
