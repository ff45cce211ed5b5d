"""What a layer in 4 bits adds to its stream, a branch at a time, by the size of the branch itself: the stream is a hundredth of
the usual one (the norms take that out), so that it does not hide what is added to it.  The formula runs in 64 bits on the
CPU over the rows that the cache holds, which are compared with their own formula; and with a mistake planted in it the layer has to be far from it."""
import math

import pytest
import torch

from brodiffusion_b200 import layer as LY
from four_bit import quantised
from test_layer4_gpu import in_4_bits, weights
from test_layer_gpu import far, rms, rotate, tables

pytestmark = pytest.mark.gpu

D, NH, NKV, HD, F = 512, 4, 2, 64, 1024
GROUP, CACHE_GROUP = 32, 64


def run(bd, w, n, window, sinks, batch, chunks, few):
    """(layer, stream, what was added to it, the cache's K and V)"""
    L = LY.FourBitLayer(w, NH, NKV, HD, window=window, sinks=sinks, group=GROUP, residual_scale=0.75)
    if few:
        L.PROMPT = L.MANY = 10 ** 9
    cos, sin = tables(512, HD)
    x = (0.01 * torch.randn(batch, n, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))).bfloat16()
    cache, parts, at = LY.KvCache4(batch, 400, NKV, HD, CACHE_GROUP, x.dtype), [], 0
    for step in chunks:
        parts.append(L.forward(x[:, at:at + step].clone(), cache, cos, sin))
        at += step
    assert at == n and bd.device_status() == 0
    k, v = (torch.empty(batch, n, NKV * HD, device="cuda", dtype=x.dtype) for _ in range(2))
    bd.cache4_read(cache.rows.first(n), k, v)
    added = torch.cat(parts, 1).double() - 0.75 ** 2 * x.double()          # (the stream is scaled ahead of each addition)
    return L, x, added.cpu(), k, v, cos, sin


def projections(L, w, x, cos, sin):
    q, k, v = (rms(x.double(), w["norm1"]) @ in_4_bits(w["wqkv"], L.group).T).split([NH * HD, NKV * HD, NKV * HD], 1)
    q, k, v = (t.view(len(x), -1, HD) for t in (q, k, v))
    return (*(rotate(rms(t, w[g]), cos[:len(x)], sin[:len(x)]) for t, g in ((q, "q_gain"), (k, "k_gain"))), v)


def attention(w, q, k, v, window, sinks, gate, post="post1"):
    """The branch from Q in 64 bits and the cache's rows, all on the CPU."""
    n = len(q)
    q, k, v = q.cpu(), *(t.cpu().double().view(n, NKV, HD).repeat_interleave(NH // NKV, 1) for t in (k, v))
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(HD)
    att = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, -math.inf), -1), v).reshape(n, -1)
    return 0.75 * rms(att @ in_4_bits(w["wo"], GROUP).cpu().T, w[post].cpu()) * gate.cpu().double()


# Roundings to BF16 are 0.0016 rms each (2^-8 / sqrt(3) / 1.4).
@pytest.mark.parametrize("n,chunks,few", [(70, [70], False), (200, [200], False), (200, [90, 1, 40, 1, 60, 8], False), (45, [20, 1, 1, 3, 20], True)])
@pytest.mark.parametrize("window,sinks", [(33, 4), (24, 0)])
def test_the_attention_branch(bd, window, sinks, n, chunks, few):
    batch, gates = 4, 2                          # a gate for every two sequences
    w, _ = weights(n, D, NH, NKV, HD, F, gates)
    w["post2"] = torch.zeros_like(w["post2"])
    L, x, added, k, v, cos, sin = run(bd, w, n, window, sinks, batch, chunks, few)
    for b in range(batch):
        qd, kd, vd = projections(L, w, x[b], cos, sin)
        for got, want in ((k[b], kd), (v[b], vd)):
            # rows of the cache: half a step, and three roundings of the values (rows, projection, norm and RoPE) and that of the row
            # read back, 2^-8 each of a group's largest; products of many rows have weights rounded to 2^-9 as well, which the
            # sum of 512 takes to 2^-9 of the root of the sum of squares, some 2^-8 of the largest
            want = want.reshape(n, -1)
            g = want.unflatten(-1, (-1, CACHE_GROUP))
            step, most = (g.amax(-1) - g.amin(-1)) / 15, g.abs().amax(-1)
            err = (got.double() - want).abs().unflatten(-1, (-1, CACHE_GROUP)).amax(-1)
            assert (err <= 0.5 * step + 8 * 2.0 ** -8 * most).all(), float(((err - 0.5 * step) / most).max())
        f = lambda window, sinks, gate=b // (batch // gates), post="post1": attention(w, qd, k[b], v[b], window, sinks, w["gate1"][gate], post)
        # rounded on the way: the rows, Q, its norm and RoPE, weights of Q (in many rows), the cache's rows read back twice, the
        # attention's weights, the heads' outputs, weights of O, the branch, the stream: eleven, of which those of Q count for a score of size
        # one: 0.0053, twice that
        want = f(window, sinks)
        assert far(added[b], want) < 0.0106, far(added[b], want)
        past = slice(window + 8, n)
        wrong = [(f(window, sinks, gate=1 - b // (batch // gates)), slice(0, n)), (f(window, sinks, post="norm1"), slice(0, n))]
        if n > window + 8:
            # a key of `window`, or a sink, less or more: sqrt(1 / window) of the rows that have as many keys, 0.16 and more
            wrong += [(f(window - 1, sinks), past), (f(window + 1, sinks), past), (f(window, sinks - 1 if sinks else 1), past)]
        for i, (t, rows) in enumerate(wrong):
            assert far(added[b][rows], t[rows]) > (0.0106 if i == 1 else 0.0212), (i, far(added[b][rows], t[rows]))


@pytest.mark.parametrize("n,chunks,few", [(1, [1], False), (40, [40], False), (200, [200], False), (61, [50, 1, 1, 9], True)])
def test_the_feed_forward_branch(bd, n, chunks, few):
    batch, gates = 2, 2
    w, _ = weights(n, D, NH, NKV, HD, F, gates)
    w["post1"] = torch.zeros_like(w["post1"])
    L, x, added, *_ = run(bd, w, n, 33, 4, batch, chunks, few)
    up, down = in_4_bits(w["w_up"], GROUP), in_4_bits(w["w_down"], GROUP)
    for b in range(batch):
        def f(act, norm="norm2", gate=b, scale=0.75):
            h = rms(scale * x[b].double(), w[norm]) @ up.T + w["b_up"].double()
            h = torch.nn.functional.silu(h) if act == "silu" else torch.nn.functional.gelu(h, approximate="tanh")
            return (rms(h @ down.T + w["b_down"].double(), w["post2"]) * w["gate2"][gate].double()).cpu()
        # rows, weights of both products (in many rows), hidden, branch, stream: six of 0.0016: 0.0039, twice that
        want = f("gelu_tanh")
        assert far(added[b], want) < 0.0078, far(added[b], want)
        for wrong in (f("silu"), f("gelu_tanh", norm="norm1"), f("gelu_tanh", gate=1 - b)):
            assert far(added[b], wrong) > 0.0156, far(added[b], wrong)


@pytest.mark.parametrize("B,n", [(4, 2), (3, 3), (3, 1), (2, 2)])
@pytest.mark.parametrize("L", [1, 2, 5])
def test_gates_of_sequences(bd, B, n, L):
    """n vectors are for B / n sequences each: the same as every sequence by itself with its own."""
    w, g = weights(B, D, NH, NKV, HD, F, n)
    cos, sin = tables(16, HD)
    x = torch.randn(B, L, D, device="cuda", generator=g).bfloat16()
    whole = LY.FourBitLayer(w, NH, NKV, HD)
    got = whole.forward(x.clone(), LY.KvCache4(B, 16, NKV, HD, 64, x.dtype), cos, sin)
    for b in range(B):
        one = LY.FourBitLayer({**w, **{k: w[k][b // (B // n)] for k in ("gate1", "gate2")}}, NH, NKV, HD)
        alone = one.forward(x[b:b + 1].clone(), LY.KvCache4(1, 16, NKV, HD, 64, x.dtype), cos, sin)
        # (products of other row counts may add up in another order: a rounding here and there, and seldom a cache's code by one)
        assert far(got[b], alone[0]) < 0.01
    assert bd.device_status() == 0
