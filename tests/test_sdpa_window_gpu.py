"""Causal attention with a sliding window and sinks against its definition in 64 bits.

Tolerance of an output value o = sum p v of n visible keys: the output's rounding, u |o|; the weights' rounding to 16
bits in front of the second product, u sum p |v|; their error from FP32 scores, exponentials and sums, below
3e-4 sum p |v| (a score of N(0, 1) rows of up to 256 columns is off by at most 256 * 2^-24 times the sum of its
products' magnitudes, 1e-4, and twice that enters a weight); FP16 weights below 2^-14 by up to 2^-25 each."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def randn(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def visible(n, lq, lk, window, sinks, key_mask):
    pos = torch.arange(n - lq, n, device="cuda")[:, None]
    key = torch.arange(lk, device="cuda")[None, :]
    seen = key <= pos
    if window:
        seen &= (pos - key < window) | (key < sinks)
    return seen if key_mask is None else seen & (key_mask != 0)


def formula(q, k, v, nh, nkv, window, sinks, lens=None, key_mask=None, scale=0.0):
    """(output, bound): q (B, Lq, nh * hd) and so on.  Masked places are left out, whatever they hold."""
    B, lq, D = q.shape
    lk, hd = k.shape[1], D // nh
    out, bound = torch.zeros(q.shape, device="cuda", dtype=torch.float64), torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    u = UNIT[q.dtype]
    for b in range(B):
        n = lk if lens is None else min(max(int(lens[b]), 0), lk)
        seen = visible(n, lq, lk, window, sinks, key_mask)
        used = seen.any(0)
        for h in range(nh):
            g = h // (nh // nkv)
            kk, vv = (torch.where(used[:, None], t[b, :, g * hd:(g + 1) * hd].double(), 0.0) for t in (k, v))
            s = q[b, :, h * hd:(h + 1) * hd].double() @ kk.T * (scale or 1 / math.sqrt(hd))
            s = s.masked_fill(~seen, -math.inf)
            p = torch.softmax(s, 1).masked_fill(~seen, 0.0)
            o = p @ vv
            out[b, :, h * hd:(h + 1) * hd] = o
            few = seen.sum(1, keepdim=True) * vv.abs().amax() * 2.0 ** -25 if q.dtype == torch.float16 else 0.0
            bound[b, :, h * hd:(h + 1) * hd] = u * o.abs() + (u + 3e-4) * (p @ vv.abs()) + few + 1e-12
    return out, bound


def call(bd, q, k, v, nh, **kw):
    out = torch.full_like(q, float("nan"))
    bd.sdpa_window_fwd(q, k, v, out, nh, **kw)
    assert bd.device_status() == 0
    return out


def check(bd, q, k, v, nh, nkv, window, sinks, lens=None, key_mask=None, scale=0.0, out=None):
    if out is None:
        kv_len = None if lens is None else torch.tensor(lens, device="cuda", dtype=torch.int32)
        out = call(bd, q, k, v, nh, window=window, sinks=sinks, num_kv_heads=nkv, kv_len=kv_len, key_mask=key_mask,
                   softmax_scale=scale)
    ref, bound = formula(q, k, v, nh, nkv, window, sinks, lens, key_mask, scale)
    err = (out.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, first {bad.nonzero()[0].tolist()}, " \
        f"worst {float((err / bound).nan_to_num(1e9).max()):.3g} times the bound"
    return out


def inputs(seed, B, lq, lk, nh, nkv, hd, dtype=torch.bfloat16):
    return randn(seed, B, lq, nh * hd, dtype=dtype), randn(seed + 1, B, lk, nkv * hd, dtype=dtype), randn(seed + 2, B, lk, nkv * hd, dtype=dtype)


# (Lq, Lk): single tokens, a few, chunks of new rows behind a cache, whole prompts, around the tile sizes
LENGTHS = [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (1, 777), (2, 130), (5, 1000), (16, 16), (17, 300), (64, 64), (65, 129), (127, 127),
           (128, 128), (129, 513), (200, 900), (257, 257), (400, 1100)]


@pytest.mark.parametrize("lq,lk", LENGTHS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (64, 4), (100, 70), (300, 0), (5000, 10)])
def test_lengths_and_windows(bd, lq, lk, window, sinks):
    q, k, v = inputs(lq * 7 + lk, 1, lq, lk, 4, 2, 64)
    check(bd, q, k, v, 4, 2, window, sinks)


@pytest.mark.parametrize("hd", [8, 40, 64, 72, 80, 128, 160, 256])
@pytest.mark.parametrize("lq,lk", [(1, 500), (3, 200), (150, 400)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_dims_and_types(bd, hd, lq, lk, dtype):
    q, k, v = inputs(hd, 2, lq, lk, 3, 3, hd, dtype)
    check(bd, q, k, v, 3, 3, 130, 20)


@pytest.mark.parametrize("nh,nkv", [(1, 1), (6, 2), (24, 8), (16, 1), (17, 1), (32, 2), (40, 1)])
@pytest.mark.parametrize("lq,lk", [(1, 700), (4, 300), (140, 333)])
def test_grouped_heads(bd, nh, nkv, lq, lk):
    q, k, v = inputs(nh, 1, lq, lk, nh, nkv, 128)
    check(bd, q, k, v, nh, nkv, 200, 8)


@pytest.mark.parametrize("lq", [1, 3, 160])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 33)])
def test_batches_of_different_lengths(bd, lq, window, sinks):
    """Lengths of zero and one, shorter than the new rows, full, and out of range (the nearer end counts); what lies
    behind a sequence's length is NaN."""
    lens = [0, 1, 2, lq, lq + 1, 64, 65, 128, 300, 511, 512, 9999, -5]
    q, k, v = inputs(lq, len(lens), lq, 512, 4, 2, 128)
    for b, n in enumerate(lens):
        k[b, max(0, n):], v[b, max(0, n):] = float("nan"), float("inf")
    out = check(bd, q, k, v, 4, 2, window, sinks, lens)
    assert (out[0] == 0).all() and (out[-1] == 0).all()


@pytest.mark.parametrize("lq,lk", [(1, 600), (2, 600), (300, 300), (260, 700)])
def test_key_masks_and_values_that_are_not_finite(bd, lq, lk):
    """Padding in front, holes, a tile and more; NaN and infinities in the masked places."""
    q, k, v = inputs(lq + lk, 2, lq, lk, 4, 4, 64)
    for kind in range(4):
        mask = torch.ones(lk, device="cuda")
        if kind == 0:
            mask[:45] = 0
        elif kind == 1:
            mask[torch.rand(lk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.5] = 0
        elif kind == 2:
            mask[100:-7] = 0
        else:
            mask[:] = 0
        kk, vv = k.clone(), v.clone()
        kk[:, mask == 0] = float("nan")
        vv[:, mask == 0] = float("inf")
        vv[:, mask == 0, ::3] = float("nan")
        out = check(bd, q, kk, vv, 4, 4, 150, 50, key_mask=mask)
        if kind == 3:
            assert (out == 0).all()
        if kind == 0 and lq == lk:
            assert (out[:, :45] == 0).all()
    check(bd, q, k, v, 4, 4, 0, 0, key_mask=torch.full((lk,), 0.25, device="cuda"))       # any factor but zero is visible


@pytest.mark.parametrize("lq,lk,bad", [(1, 400, 10), (1, 400, 250), (3, 400, 399), (140, 300, 299), (140, 300, 20)])
def test_values_outside_the_window_that_are_not_finite(bd, lq, lk, bad):
    """A key that some rows see and others do not: those that do not are as if it were not there."""
    q, k, v = inputs(bad, 1, lq, lk, 2, 1, 128)
    v[:, bad] = float("inf")
    out = call(bd, q, k, v, 2, window=100, sinks=5, num_kv_heads=1)
    seen = visible(lk, lq, lk, 100, 5, None)[:, bad]
    ref, bound = formula(q, k, torch.where(torch.isinf(v), 0.0, v), 2, 1, 100, 5)
    assert not torch.isfinite(out[0, seen]).any()
    assert ((out.double() - ref).abs() <= bound)[0, ~seen].all()


@pytest.mark.parametrize("lq", [1, 200])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(bd, lq):
    q, k, v = inputs(2, 1, lq, 300, 4, 2, 64)
    good = call(bd, q, k, v, 4, window=100, sinks=4, num_kv_heads=2)
    q[0, 0, 64:128] = float("nan")
    out = call(bd, q, k, v, 4, window=100, sinks=4, num_kv_heads=2)
    assert torch.isnan(out[0, 0, 64:128]).all()
    same = torch.ones_like(out, dtype=torch.bool)
    same[0, 0, 64:128] = False
    assert (out[same] == good[same]).all()


@pytest.mark.parametrize("lq,lk0,lk1", [(1, 100, 1), (1, 77, 300), (5, 64, 64), (130, 200, 130)])
def test_segments(bd, lq, lk0, lk1):
    """Cached rows and fresh rows as two segments, the same bits as one; the queries too."""
    nh, nkv, hd = 6, 2, 64
    q, k, v = inputs(lk0, 1, lq, lk0 + lk1, nh, nkv, hd)
    for window, sinks in ((0, 0), (60, 70), (150, 3)):
        one = check(bd, q, k, v, nh, nkv, window, sinks)
        out = torch.empty_like(q)
        bd.sdpa_window_fwd(q, [k[:, :lk0], k[:, lk0:]], [v[:, :lk0], v[:, lk0:]], out, nh, window=window, sinks=sinks, num_kv_heads=nkv)
        check(bd, q, k, v, nh, nkv, window, sinks, out=out)
        if lq > 1:
            cut = lq // 2
            outs = [torch.empty_like(q[:, :cut]), torch.empty_like(q[:, cut:])]
            bd.sdpa_window_fwd([q[:, :cut].contiguous(), q[:, cut:].contiguous()], k, v, outs, nh, window=window, sinks=sinks, num_kv_heads=nkv)
            check(bd, q, k, v, nh, nkv, window, sinks, out=torch.cat(outs, 1))
        assert torch.isfinite(one).all()


@pytest.mark.parametrize("lq", [1, 4, 140])
@pytest.mark.parametrize("hd", [64, 128])
def test_segments_with_lengths_and_a_mask(bd, lq, hd):
    """Lengths that end in either segment, masked keys in both; NaN in every place that nobody sees."""
    nh, nkv, lk0, lk1 = 4, 2, 150, 200
    lens = [0, 1, 140, 150, 151, 288, 350]
    q, k, v = inputs(hd + lq, len(lens), lq, lk0 + lk1, nh, nkv, hd)
    mask = torch.ones(lk0 + lk1, device="cuda")
    mask[20:60] = mask[145:155] = mask[300] = 0
    for t in (k, v):
        t[:, mask == 0] = float("nan")
        for b, n in enumerate(lens):
            t[b, n:] = float("nan")
    kv_len = torch.tensor(lens, device="cuda", dtype=torch.int32)
    for window, sinks in ((0, 0), (120, 30), (50, 160)):
        out = torch.empty_like(q)
        bd.sdpa_window_fwd([q], [k[:, :lk0], k[:, lk0:]], [v[:, :lk0], v[:, lk0:]], [out], nh, window=window, sinks=sinks, num_kv_heads=nkv,
                           kv_len=kv_len, key_mask=mask)
        check(bd, q, k, v, nh, nkv, window, sinks, lens, mask, out=out)


@pytest.mark.parametrize("lq", [1, 2, 150])
def test_strides(bd, lq):
    """Heads inside a wider row (a fused projection's output), a cache with room behind every sequence."""
    nh, nkv, hd, lk, B = 4, 2, 64, 190, 3
    wide = randn(1, B, lq, (nh + 2 * nkv) * hd + 24)
    cache = randn(2, B, lk + 50, 2, nkv * hd + 8)
    q, k, v = wide[:, :, 8:8 + nh * hd], cache[:, :lk, 0, :nkv * hd], cache[:, :lk, 1, :nkv * hd]
    o = torch.full((B, lq + 3, nh * hd + 40), 7.0, device="cuda", dtype=torch.bfloat16)
    bd.sdpa_window_fwd(q, k, v, o[:, :lq, 16:16 + nh * hd], nh, window=77, sinks=11, num_kv_heads=nkv)
    check(bd, q, k, v, nh, nkv, 77, 11, out=o[:, :lq, 16:16 + nh * hd])
    assert (o[:, lq:] == 7).all() and (o[:, :, :16] == 7).all() and (o[:, :, 16 + nh * hd:] == 7).all()


def test_two_dimensional_tensors_and_scale(bd):
    q, k, v = inputs(4, 1, 1, 300, 4, 4, 64)
    out = torch.empty_like(q[0])
    bd.sdpa_window_fwd(q[0], k[0], v[0], out, 4, window=50, sinks=2, softmax_scale=0.3, kv_len=torch.tensor([299], device="cuda", dtype=torch.int32))
    check(bd, q, k, v, 4, 4, 50, 2, lens=[299], scale=0.3, out=out[None])


@pytest.mark.parametrize("lq", [1, 150])
def test_large_scores(bd, lq):
    """Rows whose weights are one key's, and scores that grow along the keys (the running maximum moves at every tile)."""
    q, k, v = inputs(5, 1, lq, 700, 2, 2, 64)
    ramp = torch.linspace(0.0, 8.0, 700, device="cuda")[None, :, None]
    q2, k2 = (q.abs() * 2).to(q.dtype), (k.abs() * ramp).to(k.dtype)
    for window, sinks in ((0, 0), (300, 9)):
        out = call(bd, q2, k2, v, 2, window=window, sinks=sinks)
        ref, bound = formula(q2, k2, v, 2, 2, window, sinks)
        # scores reach 2^9: FP32 accumulation leaves each off by up to 64 * 2^-24 * 2^9 = 2e-3
        assert ((out.double() - ref).abs() <= bound + 4e-3 * v.double().abs().amax()).all()


def test_a_long_cache(bd):
    """Offsets past 2^31 elements in one sequence's cache, a single token and a chunk at its end."""
    lk, hd = 1_100_000, 128
    base = torch.zeros(lk, 2048, device="cuda", dtype=torch.bfloat16)            # 2.25e9 elements, K and V as columns of it
    k, v = base[None, :, :hd], base[None, :, hd:2 * hd]
    tail = 3000
    k[0, -tail:], v[0, -tail:] = randn(1, tail, hd), randn(2, tail, hd)
    k[0, :64], v[0, :64] = randn(3, 64, hd), randn(4, 64, hd)
    for lq in (1, 150):
        q = randn(5, 1, lq, 2 * hd)
        out = call(bd, q, k, v, 2, window=2000, sinks=60, num_kv_heads=1)
        keep = torch.cat([torch.arange(60), torch.arange(lk - tail, lk)]).cuda()
        # the same keys without the ones nobody sees: positions move, what is visible does not
        ref, bound = formula(q, k[:, keep], v[:, keep], 2, 1, 2000, 60)
        assert ((out.double() - ref).abs() <= bound).all()
    del base


def test_the_same_call_gives_the_same_bits_on_any_stream(bd):
    for lq, lk in ((1, 3000), (300, 900)):
        q, k, v = inputs(6, 2, lq, lk, 8, 2, 128)
        a = call(bd, q, k, v, 8, window=700, sinks=100, num_kv_heads=2)
        side, out = torch.cuda.Stream(), torch.empty_like(q)
        torch.cuda.synchronize()
        bd.sdpa_window_fwd(q, k, v, out, 8, window=700, sinks=100, num_kv_heads=2, stream=side)
        side.synchronize()
        assert (a == out).all()


def test_graph_follows_the_lengths(bd):
    """A captured step reads the lengths on the device: the cache grows from replay to replay."""
    q, k, v = inputs(7, 2, 1, 400, 4, 2, 64)
    out, lens = torch.empty_like(q), torch.tensor([10, 200], device="cuda", dtype=torch.int32)
    run = lambda: bd.sdpa_window_fwd(q, k, v, out, 4, window=64, sinks=4, num_kv_heads=2, kv_len=lens)
    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    for step in range(3):
        lens += 70
        g.replay()
        torch.cuda.synchronize()
        check(bd, q, k, v, 4, 2, 64, 4, lens=lens.tolist(), out=out)


def test_window_zero_is_the_causal_rule(bd):
    for lq, lk in ((1, 200), (130, 260)):
        q, k, v = inputs(8, 1, lq, lk, 4, 2, 128)
        a = call(bd, q, k, v, 4, window=0, num_kv_heads=2)
        b = torch.empty_like(q)
        bd.sdpa_fwd(q, k, v, b, 4, mask_mode=bd.MASK_CAUSAL, num_kv_heads=2)
        _, bound = formula(q, k, v, 4, 2, 0, 0)
        assert ((a.double() - b.double()).abs() <= 2 * bound).all()


def test_refusals(bd):
    q, k, v = inputs(9, 2, 3, 50, 4, 2, 64)
    out = torch.full_like(q, 7.0)
    good = dict(window=8, sinks=1, num_kv_heads=2)
    lens = torch.tensor([5, 6], device="cuda", dtype=torch.int32)
    def refuse(*args, **kw):
        with pytest.raises((bd.BdattnError, TypeError)):
            bd.sdpa_window_fwd(*args, **{**good, **kw})
    refuse(q, k, v, out, 4, window=-1)
    refuse(q, k, v, out, 4, sinks=-1)
    refuse(q, k, v, out, 4, window=1.5)
    refuse(q, k, v, out, 4, num_kv_heads=3)
    refuse(q, k, v, out, 4, kv_len=lens.long())
    refuse(q, k, v, out, 4, kv_len=lens[:1])
    refuse(q, k, v, out, 4, kv_len=[5, 6])
    refuse(q, k, v, out, 4, key_mask=torch.ones(49, device="cuda"))
    refuse(q, k, v, out, 4, key_mask=torch.ones(50, device="cuda").half())
    refuse(q, k[:1], v[:1], out, 4)
    refuse(q, k.half(), v.half(), out, 4)
    refuse(q, k, v, out[:, :2], 4)
    refuse(q.float(), k.float(), v.float(), out.float(), 4)
    refuse(q, k[:, :0], v[:, :0], out, 4)
    refuse(q[:, :, :252], k, v, out[:, :, :252], 4)                       # head_dim 63
    refuse(q[:, :, 1:], k, v, out[:, :, 1:], 4)
    p = bd.SdpaParams(dtype=bd.BF16, batch=1, num_heads=1, head_dim=64, n_q_seg=1, n_kv_seg=1, mask_mode=bd.MASK_NONE)
    w = bd.WindowParams(window=4)
    L = bd.lib()
    assert L.bdattn_sdpa_window_fwd(p, w, None) == -1 and "mask_mode" in bd.last_error()
    p.mask_mode = bd.MASK_CAUSAL
    p.key_scale = 16
    assert L.bdattn_sdpa_window_fwd(p, w, None) == -1 and "per-key scales" in bd.last_error()
    p.key_scale, p.q_cos = None, 16
    assert L.bdattn_sdpa_window_fwd(p, w, None) == -1 and "RoPE" in bd.last_error()
    p.q_cos = None
    assert L.bdattn_sdpa_window_fwd(p, w, None) == -1 and "null" in bd.last_error()
    assert L.bdattn_sdpa_window_fwd(p, None, None) == -1 and L.bdattn_sdpa_window_fwd(None, w, None) == -1
    assert (out == 7).all()
