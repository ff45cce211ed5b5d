"""A cache of K and V in 4 bits: new rows into it and back, and causal attention over it, against the formulas in 64 bits.

Rows into the cache and back are exact: the codes follow from IEEE operations, and the values are rounded once.

Tolerance of the attention, for o = sum p v with v = (low + 8 step) + step (u - 8):
  - the weights p step are rounded to FP16 once: 2^-11 of sum p step |u - 8|;
  - a score is off by at most 2^-20 of scale * sum |q| (15 step + |low|) (products exact, at most 128 of them summed by
    mma.sync, which cuts off at 2^-23, and a few FP32 steps), a weight in proportion to the scores by twice that;
  - the sums of n keys in FP32, n / 64 of them one behind the other: (n / 64 + 64) 2^-23;
  - the output is rounded once."""
import math
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from four_bit import UNIT, by_heads, flat, held, quantised, randn, values

pytestmark = pytest.mark.gpu

TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def garbage(bd, batch, heads, rows, hd, group, dtype):
    """A cache whose memory is NaN (scales) and ones (codes)."""
    c = bd.Cache4.empty(batch, heads, rows, hd, group, dtype)
    for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales):
        t.view(torch.uint8).fill_(0xff)
    return c


def bits(c):
    return [t.clone().view(torch.uint8) for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales)]


def read(bd, c, rows, kv_len=None):
    b, heads, _, half = c.k_codes.shape
    k, v = (torch.full((b, rows, heads * 2 * half), 7.0, device="cuda", dtype=c.k_scales.dtype) for _ in range(2))
    bd.cache4_read(c, k, v, kv_len=kv_len)
    assert bd.device_status() == 0
    return k, v


SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


# ------------------------------------------------------------- rows into the cache and back
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd,group", SHAPES)
@pytest.mark.parametrize("batch,heads,new,rows", [(1, 1, 1, 1), (1, 8, 1, 777), (3, 2, 5, 40), (2, 3, 129, 129), (32, 4, 1, 64)])
def test_rows_come_back_as_the_format_says(bd, batch, heads, new, rows, hd, group, dtype):
    k, v = (randn(i, batch, new, heads * hd, dtype=dtype, scale=1 + 5 * i) for i in range(2))
    c = garbage(bd, batch, heads, rows, hd, group, dtype)
    before = bits(c)
    bd.cache4_append(k, v, c)
    for got, x in zip(read(bd, c, new), (k, v)):
        assert (got == flat(held(by_heads(x, heads), group)).to(dtype)).all()
    for scales, x in ((c.k_scales, k), (c.v_scales, v)):
        assert (scales[:, :, rows - new:] == quantised(by_heads(x, heads), group)[1]).all()
    for a, b in zip(bits(c), before):                      # nothing else is written
        assert (a[:, :, :rows - new] == b[:, :, :rows - new]).all()


@pytest.mark.parametrize("new", [1, 3, 20])
def test_places_follow_the_lengths(bd, new):
    lengths = [20, 64, 0, 7, 33, 100, -5]                  # beyond the cache's 64 rows, and below 0: the nearer end
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    batch, heads, rows, hd = len(lengths), 2, 64, 64
    k, v = (randn(i, batch, new, heads * hd) for i in range(2))
    c = garbage(bd, batch, heads, rows, hd, 32, torch.bfloat16)
    before = bits(c)
    bd.cache4_append(k, v, c, kv_len=n)
    got = read(bd, c, new, n)
    for b, length in enumerate(lengths):
        length = max(0, min(rows, length))
        there = max(0, length - new)
        for x, y in zip((k, v), got):
            want = flat(held(by_heads(x[b:b + 1], heads), 32)).to(x.dtype)[0]
            lost = new - (length - there)                  # rows whose place is before the first
            assert (y[b, lost:] == want[lost:]).all() and (y[b, :lost] == 0).all()
        for a, f in zip(bits(c), before):
            assert (a[b, :, :there] == f[b, :, :there]).all() and (a[b, :, length:] == f[b, :, length:]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_groups_of_one_value_and_values_that_are_not_finite(bd, dtype):
    k = randn(1, 1, 6, 128, dtype=dtype)
    k[0, 0, :32] = 3.0                                     # step 0
    k[0, 1] = 0
    k[0, 2, 40], k[0, 3, 70], k[0, 4, 100] = float("nan"), float("inf"), -float("inf")
    k[0, 5, :32] = torch.linspace(-1, 1, 32, device="cuda").to(dtype)
    c = garbage(bd, 1, 1, 6, 128, 32, dtype)
    bd.cache4_append(k, k, c)
    for got in read(bd, c, 6):
        want = flat(held(by_heads(k, 1), 32)).to(dtype)
        assert ((got == want) | (torch.isnan(got) & torch.isnan(want))).all()
        assert int(torch.isnan(got).sum()) == 3 * 32 and (got[0, 0, :32] == 3).all() and (got[0, 1] == 0).all()


def test_a_range_beyond_fp32_counts_as_not_finite(bd):
    x = randn(1, 1, 2, 64)
    x[0, 0, 3], x[0, 0, 5] = 3e38, -3e38
    x[0, 1, 3], x[0, 1, 40] = 3e38, -3e38                  # (not in one group)
    c = garbage(bd, 1, 1, 2, 64, 32, torch.bfloat16)
    bd.cache4_append(x, x, c)
    for got in read(bd, c, 2):
        assert torch.isnan(got[0, 0, :32]).all() and torch.isfinite(got[0, 0, 32:]).all() and torch.isfinite(got[0, 1]).all()


def test_ties_and_the_ends_of_the_types(bd):
    """Quotients on the border between two codes go to the even one; the largest finite values stay finite."""
    x = torch.zeros(1, 3, 64, device="cuda", dtype=torch.float16)
    x[0, 0, :17] = torch.tensor([0.0, 15.0] + [i + 0.5 for i in range(15)], device="cuda").half()       # step 1
    x[0, 1, :4] = torch.tensor([65504.0, -65504.0, 1e-7, -3.0], device="cuda").half()
    x[0, 2, :3] = torch.tensor([6e-8, 1.2e-7, 1.8e-7], device="cuda").half()
    c = garbage(bd, 1, 1, 3, 64, 64, torch.float16)
    bd.cache4_append(x, x, c)
    got = read(bd, c, 3)[0]
    assert (got == flat(held(by_heads(x, 1), 64)).clamp(-65504, 65504).half()).all() and torch.isfinite(got).all()
    assert got[0, 0, 2:17].tolist() == [0, 2, 2, 4, 4, 6, 6, 8, 8, 10, 10, 12, 12, 14, 14]


def test_strided_rows_heads_and_items(bd):
    hd, group, heads, new = 64, 32, 3, 9
    wide = randn(1, 2, new + 4, heads * hd * 2 + 16)
    k, v = wide[:, 2:2 + new, 8:8 + heads * hd], wide[:, 1:1 + new, heads * hd + 8:2 * heads * hd + 8]
    big = garbage(bd, 5, 7, 40, hd, group, torch.bfloat16)
    part = bd.Cache4(*(getattr(big, n)[1:4:2, 2:7:2, 4:30] for n in bd.Cache4.__slots__))
    before = bits(big)
    bd.cache4_append(k, v, part)
    back = torch.full_like(wide, 5.0)
    kb, vb = back[:, 2:2 + new, 8:8 + heads * hd], torch.empty_like(v)
    bd.cache4_read(part, kb, vb)
    assert (kb == flat(held(by_heads(k, heads), group)).to(k.dtype)).all()
    assert (vb == flat(held(by_heads(v, heads), group)).to(k.dtype)).all()
    back[:, 2:2 + new, 8:8 + heads * hd] = 5.0
    assert (back == 5.0).all()
    for a, b in zip(bits(big), before):
        a[1:4:2, 2:7:2, 4 + 26 - new:30] = 0
        b[1:4:2, 2:7:2, 4 + 26 - new:30] = 0
        assert (a == b).all()
    turned = bd.Cache4(*(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (big.k_codes, big.v_codes, big.k_scales, big.v_scales)))
    bd.cache4_append(k[:, :1].expand(2, 1, -1)[:1].expand(1, 1, -1), v[:1, :1], bd.Cache4(*(getattr(turned, n)[:1, :3] for n in bd.Cache4.__slots__)))
    got = read(bd, bd.Cache4(*(getattr(turned, n)[:1, :3] for n in bd.Cache4.__slots__)), 1)
    assert (got[0] == flat(held(by_heads(k[:1, :1], heads), group)).to(k.dtype)).all()


# ------------------------------------------------------------- attention
def seen_keys(b, lq, lk, window, sinks, lengths, mask):
    """(b, lq, lk) of what is visible."""
    n = torch.tensor([max(0, min(lk, x)) for x in lengths]) if lengths is not None else torch.full((b,), lk)
    i = (n[:, None] - lq + torch.arange(lq))[:, :, None]
    j = torch.arange(lk)
    s = j <= i
    if window:
        s = s & ((j > i - window) | (j < sinks))
    if mask is not None:
        s = s & (mask.cpu() != 0)
    return s.cuda()


def check(out, q, k, v, heads, kv_heads, group, window=0, sinks=0, lengths=None, mask=None, scale=None, rows=None):
    """k, v: what was appended (b, lk, kv_heads * hd); rows that nobody sees may be anything."""
    b, lq, _ = q.shape
    lk, hd = k.shape[1], k.shape[2] // kv_heads
    scale = scale or 1 / math.sqrt(hd)
    seen = seen_keys(b, lq, lk, window, sinks, lengths, mask)
    used = seen.any(1)
    share = heads // kv_heads
    for item in range(b):
        for kv in range(kv_heads):
            on = used[item]
            see = seen[item][:, on]
            if not on.any():
                assert (out[item, :, kv * share * hd:(kv + 1) * share * hd] == 0).all()
                continue
            (kc, ks), (vc, vs) = (quantised(x[item, on, kv * hd:(kv + 1) * hd], group) for x in (k, v))
            kd, vd = values(kc, ks, group), values(vc, vs, group)
            step = vs.double().repeat_interleave(group, -2)[..., 0]
            ksize = ks.double().repeat_interleave(group, -2)
            ksize = 15 * ksize[..., 0] + ksize[..., 1].abs()
            for h in range(kv * share, (kv + 1) * share):
                qd = q[item, :, h * hd:(h + 1) * hd].double()
                s = (qd @ kd.T * scale).masked_fill(~see, -math.inf)
                p = torch.softmax(s, 1).masked_fill(~see, 0.0).nan_to_num(0.0)
                ref = p @ vd
                off = 2.0 ** -20 * scale * (qd.abs() @ ksize.T).masked_fill(~see, 0.0).amax(1, keepdim=True)
                held_ = (vd - 8 * step).abs() + 8 * step        # at least |low + 8 step| and step |u - 8|
                tol = UNIT[q.dtype] * ref.abs() + TINY[q.dtype] + (2.0 ** -11 + (lk / 64 + 64) * 2.0 ** -23) * (p @ (step * (vc - 8).abs())) + \
                    ((lk / 64 + 64) * 2.0 ** -23 + 4 * off) * (p @ held_)
                got = out[item, :, h * hd:(h + 1) * hd].double()
                err = (got - ref).abs()
                bad = ~(err <= tol) & ~(torch.isnan(got) & torch.isnan(ref))
                assert not bad.any(), f"item {item} head {h}: {int(bad.sum())} off, worst {float((err / tol).nan_to_num(99).max()):.3g} of the tolerance, rows {bad.any(1).nonzero().flatten().tolist()[:8]}"


def run(bd, q, cache, heads, **kw):
    out = torch.full_like(q, float("nan"))
    bd.sdpa_cache4_fwd(q, cache, out, heads, **kw)
    assert bd.device_status() == 0
    return out


def attend(bd, batch, lq, lk, heads, kv_heads, hd, group, dtype=torch.bfloat16, window=0, sinks=0, lengths=None, mask=None, seed=0):
    q = randn(seed, batch, lq, heads * hd, dtype=dtype)
    k = randn(seed + 1, batch, lk, kv_heads * hd, dtype=dtype) + randn(seed + 2, kv_heads * hd, dtype=dtype)
    v = randn(seed + 3, batch, lk, kv_heads * hd, dtype=dtype)
    cache = garbage(bd, batch, kv_heads, lk, hd, group, dtype)
    bd.cache4_append(k, v, cache)
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32) if lengths is not None else None
    if lengths is not None:                                # rows behind a length hold NaN
        for b, x in enumerate(lengths):
            for t in (cache.k_scales, cache.v_scales):
                t[b, :, max(0, x):] = float("nan")
    if mask is not None:
        for t in (cache.k_scales, cache.v_scales):
            t[:, :, mask == 0] = float("nan")
    out = run(bd, q, cache, heads, window=window, sinks=sinks, kv_len=n, key_mask=mask)
    check(out, q, k, v, heads, kv_heads, group, window, sinks, lengths, mask)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd,group", SHAPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 2), (16, 2), (24, 8)])
@pytest.mark.parametrize("lk", [1, 15, 16, 17, 130, 777])
def test_one_token(bd, lk, heads, kv_heads, hd, group, dtype):
    attend(bd, 1, 1, lk, heads, kv_heads, hd, group, dtype, seed=lk)


@pytest.mark.parametrize("hd,group", SHAPES)
@pytest.mark.parametrize("lq,lk", [(2, 2), (3, 50), (8, 300), (17, 17), (40, 1000), (130, 131)])
def test_several_tokens(bd, lq, lk, hd, group):
    attend(bd, 2, lq, lk, 6, 2, hd, group, seed=lq)
    attend(bd, 1, lq, lk, 3, 3, hd, group, torch.float16, seed=lq + 1)


@pytest.mark.parametrize("hd,group", [(64, 64), (128, 32)])
@pytest.mark.parametrize("lq", [1, 4, 33])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 4), (100, 33), (63, 200), (1000, 5), (0, 9)])
def test_window_and_sinks(bd, window, sinks, lq, hd, group):
    attend(bd, 2, lq, 555, 8, 2, hd, group, window=window, sinks=sinks, seed=window)


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("lq", [1, 5])
def test_lengths_and_rows_that_see_nothing(bd, lq, window):
    """Lengths of zero, one, fewer than the new rows, out of range; hidden rows hold NaN."""
    attend(bd, 8, lq, 200, 6, 2, 128, 64, window=window, sinks=3, lengths=[0, 1, 2, 16, 17, 199, 200, 150], seed=lq)
    q, kv = randn(1, 2, lq, 128), randn(2, 2, 30, 128)
    c = garbage(bd, 2, 1, 30, 128, 64, torch.bfloat16)
    bd.cache4_append(kv, kv, c)
    n = torch.tensor([-7, 1000], device="cuda", dtype=torch.int32)
    out = run(bd, q, c, 1, kv_len=n, window=window)
    check(out, q, kv, kv, 1, 1, 64, window, 0, [0, 30])
    assert (out[0] == 0).all()


@pytest.mark.parametrize("lq", [1, 6, 70])
@pytest.mark.parametrize("kind", ["start", "holes", "all", "none"])
def test_key_masks(bd, kind, lq):
    lk = 333
    j = torch.arange(lk, device="cuda")
    mask = {"start": j >= 290, "holes": j % 3 == 1, "all": j < 0, "none": j >= 0}[kind].float()
    out = attend(bd, 2, lq, lk, 4, 2, 64, 32, torch.float16, window=100, sinks=7, mask=mask, seed=lq)
    if kind == "all":
        assert (out == 0).all()


def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(bd):
    """One key's values are NaN: the queries behind it are NaN, those ahead of it are not."""
    lq, lk, hd = 12, 60, 64
    q, k, v = randn(1, 1, lq, 2 * hd), randn(2, 1, lk, hd), randn(3, 1, lk, hd)
    for where in ("v", "k"):
        kk, vv = k.clone(), v.clone()
        (vv if where == "v" else kk)[0, 53, :32] = float("nan")
        c = garbage(bd, 1, 1, lk, hd, 32, torch.bfloat16)
        bd.cache4_append(kk, vv, c)
        out = run(bd, q, c, 2)
        first = 53 - (lk - lq)                             # the first query that sees it
        check(out[:, :first], q[:, :first], k[:, :lk - lq + first], v[:, :lk - lq + first], 2, 1, 32)
        bad = torch.isnan(out[0, first:].view(-1, 2, hd))
        assert (bad[..., :32] if where == "v" else bad).all()
        if where == "v":
            assert not bad[..., 32:].any()


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e-20), (torch.bfloat16, 1e20), (torch.float16, 1e-3), (torch.float16, 50.0), (torch.float16, 500.0)])
def test_magnitudes_of_values(bd, dtype, size):
    """Steps of V of any size, and of very different sizes from key to key.  (500 * 2^8 is beyond FP16 from half a standard
    deviation on: groups with an infinity, which are NaN, in the formula as in the output.)"""
    q, k, v = randn(1, 1, 2, 256, dtype=dtype), randn(2, 1, 400, 128, dtype=dtype), randn(3, 1, 400, 128, dtype=torch.float32)
    v = (v * size * 2.0 ** (torch.arange(400, device="cuda") % 9)[:, None]).to(dtype)
    c = garbage(bd, 1, 1, 400, 128, 32, dtype)
    bd.cache4_append(k, v, c)
    check(run(bd, q, c, 2), q, k, v, 2, 1, 32)


@pytest.mark.parametrize("dtype,q_size,k_size", [(torch.bfloat16, 1e15, 1e-15), (torch.bfloat16, 1e-20, 1e20), (torch.float16, 1e-4, 1e4), (torch.float16, 1e4, 1e-3)])
def test_magnitudes_of_queries_and_keys(bd, dtype, q_size, k_size):
    q, k = (randn(i, 1, 2, 256, dtype=torch.float32) for i in range(2)), None
    q = (next(q) * q_size).to(dtype)
    k, v = (randn(5, 1, 400, 128, dtype=torch.float32) * k_size).to(dtype), randn(6, 1, 400, 128, dtype=dtype)
    c = garbage(bd, 1, 1, 400, 128, 64, dtype)
    bd.cache4_append(k, v, c)
    check(run(bd, q, c, 2), q, k, v, 2, 1, 64)


@pytest.mark.parametrize("q_size,scale", [(1e37, 0.0), (1e-30, 1e-30), (1.0, 1e-38)])
def test_factors_beyond_fp32(bd, q_size, scale):
    """The factor of the scores passes FP32's ends: the largest score takes all, or all seen keys count alike; hidden ones count for
    nothing."""
    q, k, v = randn(1, 1, 3, 128, scale=q_size), randn(2, 1, 100, 128), randn(3, 1, 100, 128)
    c = garbage(bd, 1, 1, 100, 128, 64, torch.bfloat16)
    bd.cache4_append(k, v, c)
    out = torch.empty_like(q)
    bd.sdpa_cache4_fwd(q, c, out, 1, softmax_scale=scale)
    kh, vh = held(k, 64)[0], held(v, 64)[0]
    for i in range(3):
        n = 98 + i
        want = vh[(kh[:n] @ q[0, i].double()).argmax()] if scale == 0 else vh[:n].mean(0)
        # (a weight times a step and the output are rounded once each, and 2^-11 is the more for the FP32 sums)
        bound = 2.0 ** -8 * want.abs() + 2.0 ** -11 * vh[:n].abs().amax(0)
        assert ((out[0, i].double() - want).abs() <= bound).all()


def test_queries_of_zeros_and_a_scale(bd):
    q, k, v = randn(1, 1, 3, 256), randn(2, 1, 100, 128), randn(3, 1, 100, 128)
    q[0, 1] = 0
    c = garbage(bd, 1, 1, 100, 128, 128, torch.bfloat16)
    bd.cache4_append(k, v, c)
    check(run(bd, q, c, 2, softmax_scale=0.5), q, k, v, 2, 1, 128, scale=0.5)


@pytest.mark.parametrize("batch,lk", [(1, 5000), (7, 3001), (40, 700), (1, 33000)])
def test_long_caches(bd, batch, lk):
    lengths = [lk - 97 * b for b in range(batch)]
    attend(bd, batch, 1, lk, 4, 2, 128, 32, lengths=lengths if batch > 1 else None, seed=batch)
    attend(bd, batch, 3, lk, 4, 2, 64, 64, torch.float16, seed=batch + 1)


def test_offsets_beyond_32_bits(bd):
    rows, hd, lq = 36_000_000, 128, 2                      # 2.3 GB of codes
    c = bd.Cache4.empty(1, 1, rows, hd, 128, torch.bfloat16)
    k, v, q = randn(1, 1, 300, hd), randn(2, 1, 300, hd), randn(3, 1, lq, 2 * hd)
    bd.cache4_append(k, v, c)
    got = read(bd, c, 300)
    assert (got[0] == flat(held(by_heads(k, 1), 128)).to(k.dtype)).all() and (got[1] == flat(held(by_heads(v, 1), 128)).to(k.dtype)).all()
    out = run(bd, q, c, 2, window=250)
    check(out, q, k, v, 2, 1, 128, window=250)
    many = garbage(bd, 600, 2, 65536, 64, 64, torch.bfloat16)          # items beyond 2^31 bytes
    kk = randn(4, 600, 1, 128)
    n = torch.full((600,), 20, device="cuda", dtype=torch.int32)
    bd.cache4_append(kk, kk, many, kv_len=n)
    assert (read(bd, many, 1, n)[0] == flat(held(by_heads(kk, 2), 64)).to(kk.dtype)).all()
    out = run(bd, kk, many, 2, kv_len=n, window=1)
    assert (out == read(bd, many, 1, n)[1]).all()          # the own key alone is seen


def test_strided_queries_and_cache(bd):
    hd, group, lq, lk = 64, 32, 5, 90
    wide = randn(1, 2, lq + 3, 6 * hd + 24)
    q = wide[:, 1:1 + lq, 16:16 + 6 * hd]
    big = garbage(bd, 4, 5, 128, hd, group, torch.bfloat16)
    part = bd.Cache4(*(getattr(big, n)[::2, 1:5:2, :lk] for n in bd.Cache4.__slots__))
    k, v = randn(2, 2, lk, 2 * hd), randn(3, 2, lk, 2 * hd)
    bd.cache4_append(k, v, part)
    full = torch.full_like(wide, 5.0)
    out = full[:, 2:2 + lq, 8:8 + 6 * hd]
    bd.sdpa_cache4_fwd(q, part, out, 6)
    check(out, q, k, v, 6, 2, group)
    full[:, 2:2 + lq, 8:8 + 6 * hd] = 5.0
    assert (full == 5.0).all()


def test_the_same_call_gives_the_same_bits_on_any_stream_and_captured(bd):
    q, k, v = randn(1, 2, 4, 512), randn(2, 2, 900, 256), randn(3, 2, 900, 256)
    c = garbage(bd, 2, 2, 1000, 128, 32, torch.bfloat16)
    n = torch.tensor([900, 900], device="cuda", dtype=torch.int32)
    bd.cache4_append(k, v, c, kv_len=n)
    want = run(bd, q, c, 4, kv_len=n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = run(bd, q, c, 4, kv_len=n, stream=side)
    side.synchronize()
    assert (out == want).all()
    # a captured step follows the lengths: the new rows' places and what is seen
    k1, v1 = randn(4, 2, 4, 256), randn(5, 2, 4, 256)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bd.cache4_append(k1, v1, c, kv_len=n)
        bd.sdpa_cache4_fwd(q, c, out, 4, kv_len=n)
    n += 4
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        k, v = torch.cat([k, k1], 1), torch.cat([v, v1], 1)
        check(out, q, k, v, 4, 2, 32)
        k1.copy_(randn(6, 2, 4, 256))
        n += 4


@pytest.mark.parametrize("lq,hd,window", [(1, 128, 0), (3, 64, 40), (70, 64, 0)])
def test_the_output_in_the_queries_place(bd, lq, hd, window):
    q, k, v = randn(1, 2, lq, 4 * hd), randn(2, 2, 3000, 2 * hd), randn(3, 2, 3000, 2 * hd)
    c = garbage(bd, 2, 2, 3000, hd, 32, torch.bfloat16)
    bd.cache4_append(k, v, c)
    apart = run(bd, q, c, 4, window=window)
    bd.sdpa_cache4_fwd(q, c, q, 4, window=window)
    assert torch.equal(q, apart)


def test_calls_at_once(bd):
    """Two host threads with a stream and tensors of their own each: the bits of calls one behind the other."""
    def work(i, stream):
        heads, hd = (4, 128) if i else (8, 64)
        q, k, v = randn(i, 3, 2, heads * hd), randn(i + 2, 3, 5000, heads * hd // 2), randn(i + 4, 3, 5000, heads * hd // 2)
        packed = torch.randint(0, 100, (bd.w4_bytes(1291, heads * hd, 64),), device="cuda", dtype=torch.uint8, generator=torch.Generator("cuda").manual_seed(i))
        x, res = q.view(6, -1), randn(i + 6, 6, heads * hd)
        c = garbage(bd, 3, heads // 2, 5000, hd, 64, torch.bfloat16)
        out = []
        stream.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            bd.cache4_append(k, v, c, stream=stream)
            with torch.cuda.stream(stream):
                o, y, r = torch.empty_like(q), torch.empty(6, 1291, device="cuda", dtype=torch.bfloat16), torch.empty_like(res)
            bd.sdpa_cache4_fwd(q, c, o, heads, stream=stream)
            bd.linear_w4_fwd(x, packed, None, y, group=64, stream=stream)
            bd.sandwich_norm_fwd(x, res, r, stream=stream)
            out.append((o, y, r))
        stream.synchronize()
        return out
    streams = [torch.cuda.Stream() for _ in range(2)]
    alone = [work(i, s)[0] for i, s in enumerate(streams)]
    with ThreadPoolExecutor(2) as pool:
        together = [f.result() for f in [pool.submit(work, i, s) for i, s in enumerate(streams)]]
    for one, many in zip(alone, together):
        for got in many:
            for a, b in zip(one, got):
                assert torch.equal(a.view(torch.int16), b.view(torch.int16))


CAPTURED_FIRST = """
import torch, brodiffusion_b200 as bd
r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
q, k, x = r(1, 1, 1024), r(1, 32768, 1024), r(40, 1024)
c = bd.Cache4.empty(1, 8, 32768, 128, 32, torch.bfloat16)
w = torch.zeros(bd.w4_bytes(5000, 1024, 32), device="cuda", dtype=torch.uint8)
o, y, m, t = torch.empty_like(q), torch.empty(40, 5000, device="cuda", dtype=torch.bfloat16), r(5000, 1024), torch.empty_like(x)
calls = lambda: (bd.cache4_append(k, k, c), bd.sdpa_cache4_fwd(q, c, o, 8), bd.linear_w4_fwd(x, w, None, y, group=32), bd.w4_unpack(w, m, group=32),
                 bd.sandwich_norm_fwd(x, x, t))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls()
g.replay()
torch.cuda.synchronize()
first = [a.clone() for a in (o, y, m, t)]
calls()
assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(first, (o, y, m, t))) and bd.device_status() == 0
print("captured first")
"""


def test_a_processs_first_calls_are_captured():
    """What a launch looks up once (limits of shared memory, clusters of more than eight CTAs) is no obstacle to a capture."""
    res = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], capture_output=True, text=True, timeout=300,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert res.returncode == 0 and "captured first" in res.stdout, res.stderr[-2000:]


def test_refusals(bd):
    c = bd.Cache4.empty(2, 2, 64, 64, 32, torch.bfloat16)
    q, k = randn(1, 2, 3, 256), randn(2, 2, 3, 128)
    out, n = torch.empty_like(q), torch.tensor([5, 6], device="cuda", dtype=torch.int32)
    other = lambda **kw: bd.Cache4(*(kw.get(s, getattr(c, s)) for s in bd.Cache4.__slots__))
    for call in (lambda: bd.cache4_append(k, k[:1], c),
                 lambda: bd.cache4_append(k[:1], k[:1], c),
                 lambda: bd.cache4_append(k[..., :64], k[..., :64], c),
                 lambda: bd.cache4_append(k.half(), k.half(), c),
                 lambda: bd.cache4_append(k, k.half(), c),
                 lambda: bd.cache4_append(k, k, c, kv_len=n.long()),
                 lambda: bd.cache4_append(k, k, c, kv_len=n[:1]),
                 lambda: bd.cache4_append(k[..., 4:], k[..., 4:], c),
                 lambda: bd.cache4_append(k, k, other(k_codes=c.k_codes[..., :16])),
                 lambda: bd.cache4_append(k, k, other(k_codes=c.k_codes.view(torch.int8))),
                 lambda: bd.cache4_append(k, k, other(v_scales=c.v_scales.half())),
                 lambda: bd.cache4_append(k, k, other(v_scales=c.v_scales[:, :, :, :1])),
                 lambda: bd.cache4_append(k, k, bd.Cache4(*(getattr(c, s)[:, :, ::2] for s in bd.Cache4.__slots__))),
                 lambda: bd.cache4_append(k, k, bd.Cache4(*(getattr(c, s)[:1].expand(2, -1, -1, *([-1] * (getattr(c, s).dim() - 3))) for s in bd.Cache4.__slots__))),
                 lambda: bd.cache4_append(k, k, bd.Cache4.empty(2, 1, 64, 128, 8, torch.bfloat16)),          # groups of 8
                 lambda: bd.cache4_read(c, k, k[:, :2]),
                 lambda: bd.sdpa_cache4_fwd(q, c, out, 3),
                 lambda: bd.sdpa_cache4_fwd(q, c, out, 0),
                 lambda: bd.sdpa_cache4_fwd(q, c, out[:, :2], 4),
                 lambda: bd.sdpa_cache4_fwd(q[:1], c, out[:1], 4),
                 lambda: bd.sdpa_cache4_fwd(q.half(), c, out.half(), 4),
                 lambda: bd.sdpa_cache4_fwd(q, c, out, 4, window=-1),
                 lambda: bd.sdpa_cache4_fwd(q, c, out, 4, sinks=-1),
                 lambda: bd.sdpa_cache4_fwd(q, c, out, 4, key_mask=torch.ones(63, device="cuda")),
                 lambda: bd.sdpa_cache4_fwd(q, c, out, 4, key_mask=torch.ones(64, device="cuda").half()),
                 lambda: bd.sdpa_cache4_fwd(q[:, :0], c, out[:, :0], 4),
                 lambda: bd.sdpa_cache4_fwd(q[..., :192].contiguous(), c, out[..., :192].contiguous(), 3)):    # 3 heads over 2
        with pytest.raises(bd.BdattnError):
            call()
    bd.cache4_append(k[:, :0], k[:, :0], c)                # no rows: nothing is done
    good = dict(dtype=bd.BF16, batch=2, num_kv_heads=2, head_dim=64, group=32, rows=64, k_codes=c.k_codes.data_ptr(), v_codes=c.v_codes.data_ptr(),
                k_scales=c.k_scales.data_ptr(), v_scales=c.v_scales.data_ptr())
    r = bd.Cache4Rows(rows=3, k=k.data_ptr(), v=k.data_ptr())
    for change, reason in ((dict(dtype=bd.F32), "dtype"), (dict(head_dim=96), "head_dim"), (dict(group=128), "group"), (dict(rows=0), "rows"),
                           (dict(k_codes=0), "null"), (dict(codes_head_stride=1024), "overlap"), (dict(codes_batch_stride=2048), "overlap"),
                           (dict(codes_head_stride=2056), "16"), (dict(k_scales=c.k_scales.data_ptr() + 4), "aligned"),
                           (dict(scales_head_stride=258), "aligned"), (dict(batch=0), "batch"), (dict(num_kv_heads=70000), "batch")):
        p = bd.Cache4Params(**{**good, **change})
        assert bd.lib().bdattn_cache4_append(p, r, None) == -1 and reason in bd.last_error(), (change, bd.last_error())
    p = bd.Cache4Params(**good)
    for change, reason in ((dict(rows=-1), "rows"), (dict(k=0), "null"), (dict(k_ld=64), "stride"), (dict(k_ld=132), "multiples"),
                           (dict(kv_len=n.data_ptr() + 1), "aligned")):
        r2 = bd.Cache4Rows(**{**dict(rows=3, k=k.data_ptr(), v=k.data_ptr()), **change})
        assert bd.lib().bdattn_cache4_append(p, r2, None) == -1 and reason in bd.last_error(), (change, bd.last_error())
    a = bd.SdpaCache4Params(num_heads=4, q_rows=1 << 30, q=q.data_ptr(), o=out.data_ptr())
    assert bd.lib().bdattn_sdpa_cache4_fwd(p, a, None) == -1 and "2^30" in bd.last_error()
    assert bd.lib().bdattn_sdpa_cache4_fwd(p, None, None) == -1 and bd.lib().bdattn_sdpa_cache4_fwd(None, a, None) == -1
