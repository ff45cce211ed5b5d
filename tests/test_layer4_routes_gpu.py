"""The attention of a layer in 4 bits by way of 16-bit rows reads back no more than its window shows; the same stream whichever
way it takes."""
import pytest
import torch

import brodiffusion_b200 as bd_
from brodiffusion_b200 import layer as LY
from test_layer4_gpu import BOUND, weights
from test_layer_gpu import far, tables

pytestmark = pytest.mark.gpu


def stream(bd, monkeypatch, L, x, filled, prompt, nkv, hd, lk):
    """Prompts of their own lengths, then x's new tokens; (what x becomes, the rows that cache4_read was asked for)."""
    cos, sin = tables(lk, hd)
    cache = LY.KvCache4(len(filled), lk, nkv, hd, 64, x.dtype)
    for t in (cache.rows.k_scales, cache.rows.v_scales):
        t.fill_(float("nan"))
    for b, n in enumerate(filled):
        one = LY.KvCache4(1, lk, nkv, hd, 64, x.dtype)
        one.rows = bd.Cache4(*(getattr(cache.rows, s)[b:b + 1] for s in bd.Cache4.__slots__))
        g = torch.Generator("cuda").manual_seed(b)
        L.forward(torch.randn(1, n, x.shape[2], device="cuda", generator=g).bfloat16(), one, cos, sin)
        cache.filled[b] = n
    cache.lengths.copy_(torch.tensor(filled, dtype=torch.int32))
    asked, read = [], bd_.cache4_read

    def counted(held, k, v, **kw):
        asked.append(k.shape[1])
        read(held, k, v, **kw)
    with monkeypatch.context() as m:
        m.setattr(bd_, "cache4_read", counted)
        m.setattr(LY.FourBitLayer, "PROMPT", prompt)
        got = L.forward(x.clone(), cache, cos, sin)
    assert bd.device_status() == 0 and cache.filled == [n + x.shape[1] for n in filled]
    return got, asked


@pytest.mark.parametrize("window,sinks,new,filled,rows", [
    (40, 0, 33, [200, 200], [72]), (40, 5, 64, [300, 151, 230], [5, 103]), (16, 3, 40, [18, 500], [3, 55]), (40, 5, 33, [44, 90], [5, 72]),
    (40, 5, 33, [43, 90], [123]),                  # (a row short in one sequence: all of them)
    (500, 5, 40, [100, 90], [140]), (0, 0, 40, [100, 90], [140])])
def test_rows_that_are_read_back(bd, monkeypatch, window, sinks, new, filled, rows):
    D, nh, nkv, hd, F = 512, 6, 2, 64, 512
    w, g = weights(new, D, nh, nkv, hd, F, 0)
    L = LY.FourBitLayer(w, nh, nkv, hd, window=window, sinks=sinks)
    x = torch.randn(len(filled), new, D, device="cuda", generator=g).bfloat16()
    by_rows, asked = stream(bd, monkeypatch, L, x, filled, 32, nkv, hd, 600)
    assert asked == rows
    by_codes, asked = stream(bd, monkeypatch, L, x, filled, 10 ** 9, nkv, hd, 600)
    assert asked == []
    # the caches are the same to the bit, so what differs is K and V in 16 bits, 0.0016 rms of each, and the roundings of the steps behind
    # (eight of them, of as much: 0.0046, twice that)
    assert far(by_rows, by_codes) < 0.01 < BOUND
