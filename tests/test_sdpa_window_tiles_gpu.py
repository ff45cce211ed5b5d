"""Windowed attention on the tensor-core kernel: calls with more than 64 rows to a K/V head and more sixteens of rows
than the GPU has SMs, which go to no other.  Same definition and bounds as tests/test_sdpa_window_gpu.py."""
import pytest
import torch

import test_sdpa_window_gpu as W

pytestmark = pytest.mark.gpu


def tiles(B, lq, nh, nkv):
    """Asserts that the call is one of the tensor-core kernel's."""
    rows = lq * (nh // nkv)
    assert rows > 64 and B * nkv * -(-rows // 16) > torch.cuda.get_device_properties(0).multi_processor_count
    return W


@pytest.mark.parametrize("lq,lk", [(65, 65), (65, 129), (127, 127), (128, 128), (129, 513), (200, 900), (256, 256), (257, 257), (400, 1100)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (64, 4), (100, 70), (128, 128), (300, 0), (300, 150), (5000, 10)])
@pytest.mark.parametrize("hd", [64, 128])
def test_lengths_and_windows(bd, lq, lk, window, sinks, hd):
    nh = 32
    q, k, v = W.inputs(lq * 7 + lk, 1, lq, lk, nh, nh, hd)
    tiles(1, lq, nh, nh).check(bd, q, k, v, nh, nh, window, sinks)


@pytest.mark.parametrize("hd", [8, 40, 64, 72, 80, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_dims_and_types(bd, hd, dtype):
    q, k, v = W.inputs(hd, 2, 150, 400, 12, 12, hd, dtype)
    tiles(2, 150, 12, 12).check(bd, q, k, v, 12, 12, 130, 20)


@pytest.mark.parametrize("nh,nkv", [(24, 8), (32, 2), (40, 1)])
def test_grouped_heads(bd, nh, nkv):
    q, k, v = W.inputs(nh, 2, 140, 333, nh, nkv, 128)
    tiles(2, 140, nh, nkv).check(bd, q, k, v, nh, nkv, 200, 8)


@pytest.mark.parametrize("B,lq", [(16, 70), (13, 160), (3, 513)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 33)])
@pytest.mark.parametrize("hd", [64, 128])
def test_batches_of_different_lengths(bd, B, lq, window, sinks, hd):
    """Lengths of zero and one, shorter than the new rows, full and out of range; NaN and infinities behind them."""
    lens = ([0, 1, 2, lq, lq + 1, 64, 65, 128, 300, 511, 512, 9999, -5, 129, 127, 256] * 2)[:B]
    q, k, v = W.inputs(lq, B, lq, 600, 8, 4, hd)
    for b, n in enumerate(lens):
        k[b, max(0, n):], v[b, max(0, n):] = float("nan"), float("inf")
    out = tiles(B, lq, 8, 4).check(bd, q, k, v, 8, 4, window, sinks, lens)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("lq,lk", [(300, 300), (130, 700)])
@pytest.mark.parametrize("hd", [64, 128])
def test_key_masks_and_values_that_are_not_finite(bd, lq, lk, hd):
    nh = 24
    q, k, v = W.inputs(lq + lk, 1, lq, lk, nh, nh, hd)
    for kind in range(5):
        mask = torch.ones(lk, device="cuda")
        if kind == 0:
            mask[:140] = 0                                        # a whole tile and more in front
        elif kind == 1:
            mask[torch.rand(lk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.5] = 0
        elif kind == 2:
            mask[100:-7] = 0
        elif kind == 3:
            mask[128:256] = 0                                     # a tile in between
        else:
            mask[:] = 0
        kk, vv = k.clone(), v.clone()
        kk[:, mask == 0] = float("nan")
        vv[:, mask == 0] = float("inf")
        vv[:, mask == 0, ::3] = float("nan")
        for window, sinks in ((150, 50), (0, 0)):
            tiles(1, lq, nh, nh).check(bd, q, kk, vv, nh, nh, window, sinks, key_mask=mask)


@pytest.mark.parametrize("bad", [299, 20, 150])
@pytest.mark.parametrize("hd", [64, 128])
def test_values_outside_the_window_that_are_not_finite(bd, bad, hd):
    nh, lq, lk = 40, 140, 300
    q, k, v = W.inputs(bad, 1, lq, lk, nh, nh, hd)
    v[:, bad] = float("inf")
    tiles(1, lq, nh, nh)
    out = W.call(bd, q, k, v, nh, window=100, sinks=5)
    seen = W.visible(lk, lq, lk, 100, 5, None)[:, bad]
    ref, bound = W.formula(q, k, torch.where(torch.isinf(v), 0.0, v), nh, nh, 100, 5)
    assert not torch.isfinite(out[0, seen]).any()
    assert ((out.double() - ref).abs() <= bound)[0, ~seen].all()


def test_a_query_that_is_not_finite_spoils_its_own_row_only(bd):
    nh, lq = 24, 200
    q, k, v = W.inputs(2, 1, lq, 300, nh, nh, 64)
    tiles(1, lq, nh, nh)
    good = W.call(bd, q, k, v, nh, window=100, sinks=4)
    q[0, 0, 64:128] = float("nan")
    out = W.call(bd, q, k, v, nh, window=100, sinks=4)
    assert torch.isnan(out[0, 0, 64:128]).all()
    same = torch.ones_like(out, dtype=torch.bool)
    same[0, 0, 64:128] = False
    assert (out[same] == good[same]).all()


def test_segments_with_lengths_and_a_mask(bd):
    nh, lq, lk0, lk1, hd = 16, 140, 150, 200, 128
    lens = [0, 1, 140, 150, 151, 288, 350]
    q, k, v = W.inputs(1, len(lens), lq, lk0 + lk1, nh, nh, hd)
    mask = torch.ones(lk0 + lk1, device="cuda")
    mask[20:60] = mask[145:155] = mask[300] = 0
    for t in (k, v):
        t[:, mask == 0] = float("nan")
        for b, n in enumerate(lens):
            t[b, n:] = float("nan")
    kv_len = torch.tensor(lens, device="cuda", dtype=torch.int32)
    tiles(len(lens), lq, nh, nh)
    for window, sinks in ((0, 0), (120, 30), (50, 160)):
        for m in (None, mask):
            out = torch.empty_like(q)
            kk, vv = (k, v) if m is not None else (torch.where(torch.isnan(k), 0.5, k), torch.where(torch.isnan(v), 0.5, v))
            bd.sdpa_window_fwd([q], [kk[:, :lk0], kk[:, lk0:]], [vv[:, :lk0], vv[:, lk0:]], [out], nh, window=window, sinks=sinks,
                               kv_len=kv_len, key_mask=m)
            W.check(bd, q, kk, vv, nh, nh, window, sinks, lens, m, out=out)


def test_strides(bd):
    nh, nkv, hd, lk, B, lq = 12, 6, 64, 190, 3, 150
    wide = W.randn(1, B, lq, (nh + 2 * nkv) * hd + 24)
    cache = W.randn(2, B, lk + 50, 2, nkv * hd + 8)
    q, k, v = wide[:, :, 8:8 + nh * hd], cache[:, :lk, 0, :nkv * hd], cache[:, :lk, 1, :nkv * hd]
    o = torch.full((B, lq + 3, nh * hd + 40), 7.0, device="cuda", dtype=torch.bfloat16)
    tiles(B, lq, nh, nkv)
    bd.sdpa_window_fwd(q, k, v, o[:, :lq, 16:16 + nh * hd], nh, window=77, sinks=11, num_kv_heads=nkv)
    W.check(bd, q, k, v, nh, nkv, 77, 11, out=o[:, :lq, 16:16 + nh * hd])
    assert (o[:, lq:] == 7).all() and (o[:, :, :16] == 7).all() and (o[:, :, 16 + nh * hd:] == 7).all()


def test_large_scores(bd):
    nh, lq = 24, 150
    q, k, v = W.inputs(5, 1, lq, 700, nh, nh, 64)
    ramp = torch.linspace(0.0, 8.0, 700, device="cuda")[None, :, None]
    q2, k2 = (q.abs() * 2).to(q.dtype), (k.abs() * ramp).to(k.dtype)
    tiles(1, lq, nh, nh)
    for window, sinks in ((0, 0), (300, 9)):
        out = W.call(bd, q2, k2, v, nh, window=window, sinks=sinks)
        ref, bound = W.formula(q2, k2, v, nh, nh, window, sinks)
        assert ((out.double() - ref).abs() <= bound + 4e-3 * v.double().abs().amax()).all()


def test_a_long_cache(bd):
    """Offsets past 2^31 elements, and more key tiles than a list of them has numbers for."""
    lk, hd, nh, lq = 4_300_000, 64, 32, 100
    base = torch.zeros(lk, 2 * hd + 384, device="cuda", dtype=torch.bfloat16)            # 2.2e9 elements
    k, v = base[None, :, :hd], base[None, :, hd:2 * hd]
    tail = 3000
    k[0, -tail:], v[0, -tail:] = W.randn(1, tail, hd), W.randn(2, tail, hd)
    k[0, :64], v[0, :64] = W.randn(3, 64, hd), W.randn(4, 64, hd)
    q = W.randn(5, 1, lq, nh * hd)
    tiles(1, lq, nh, 1)
    keep = torch.cat([torch.arange(60), torch.arange(lk - tail, lk)]).cuda()
    for mask in (None, torch.ones(lk, device="cuda")):
        if mask is not None:
            mask[lk - 500:lk - 400] = 0
        out = W.call(bd, q, k, v, nh, window=2000, sinks=60, num_kv_heads=1, key_mask=mask)
        ref, bound = W.formula(q, k[:, keep], v[:, keep], nh, 1, 2000, 60, key_mask=None if mask is None else mask[keep])
        assert ((out.double() - ref).abs() <= bound).all()
    del base
