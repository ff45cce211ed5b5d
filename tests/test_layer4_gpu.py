"""A causal layer with weights and cache in 4 bits (brodiffusion_b200/layer.py: FourBitLayer) against its steps in 64 bits, and
its calls against one another: a prompt at once, in chunks and token by token."""
import math

import pytest
import torch

from brodiffusion_b200 import layer as LY
from four_bit import by_heads, flat, held, quantised, values
from test_layer_gpu import far, make, rms, rotate, tables

pytestmark = pytest.mark.gpu


def weights(seed, D, nh, nkv, hd, F, gates, gains=True):
    w, g = make(seed, D, nh, nkv, hd, F, gains=gains)
    r = lambda *s, scale: (scale * torch.randn(*s, device="cuda", generator=g)).bfloat16()
    w.update(post1=1 + r(D, scale=0.02), post2=1 + r(D, scale=0.02))
    if gates:
        w.update(gate1=1 + r(gates, D, scale=0.3), gate2=1 + r(gates, D, scale=0.3))
    return w, g


def in_4_bits(w, group):
    """The values that the layer holds of a matrix."""
    cols = w.shape[1]
    whole = -(-cols // group) * group
    codes, scales = quantised(torch.cat([w, w[:, -1:].expand(-1, whole - cols)], 1), group)
    return values(codes[:, :cols], scales, group)


def formula(L, w, stream, cos, sin, gate, cache_group):
    """One sequence from its start, all steps in 64 bits; the cache's rows as it holds them (of K and V rounded to 16 bits)."""
    nh, nkv, hd, n = L.nh, L.nkv, L.hd, stream.shape[0]
    m = {name: in_4_bits(w[name], L.group) for name in ("wqkv", "wo", "w_up", "w_down")}
    x = stream.double()
    q, k, v = (rms(x, w["norm1"]) @ m["wqkv"].T).split([nh * hd, nkv * hd, nkv * hd], 1)
    q, k, v = (t.view(n, -1, hd) for t in (q, k, v))
    q = rotate(rms(q, w.get("q_gain")) if "q_gain" in w else q, cos[:n], sin[:n])
    k = rotate(rms(k, w.get("k_gain")) if "k_gain" in w else k, cos[:n], sin[:n])
    k, v = (held(t.bfloat16(), cache_group).repeat_interleave(nh // nkv, 1) for t in (k, v))
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    seen = (j <= i) & ((i - j < L.window) | (j < L.sinks)) if L.window else j <= i
    s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd)
    att = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, -math.inf), -1), v).reshape(n, -1)
    x = L.scale * x + rms(att @ m["wo"].T, w["post1"]) * (gate["gate1"].double() if gate else 1)
    h = torch.nn.functional.gelu(rms(x, w["norm2"]) @ m["w_up"].T + w["b_up"].double(), approximate="tanh")
    return L.scale * x + rms(h @ m["w_down"].T + w["b_down"].double(), w["post2"]) * (gate["gate2"].double() if gate else 1)


# What stands between the steps is rounded to 16 bits, 2^-9 rms of each: seven of them in a row of the branches; and K and V so
# rounded fall on another code where they were near the border of two: 2^-9 of the value is up to a tenth of a step (of a
# fifteenth of a group's range, some five times the values' root mean square), a tenth of the codes by one step each:
# 0.1^0.5 * 5 / 15 = 0.1 of a value, of which the softmax of n keys leaves n^-0.5 of its own size, that is the branch's; the norm
# behind the branch keeps the proportion.  Half of that stays in the second branch.  0.1 of branches of the stream's size.
BOUND = 0.1


@pytest.mark.parametrize("D,nh,nkv,hd,F,n,group,cache_group", [(512, 4, 2, 64, 1024, 200, 32, 32), (640, 6, 2, 128, 1288, 33, 128, 64),
                                                               (1280, 8, 8, 64, 2560, 7, 64, 64)])
@pytest.mark.parametrize("window,sinks,gates", [(0, 0, 0), (64, 4, 2)])
def test_a_prompt_against_the_formulas(bd, D, nh, nkv, hd, F, n, group, cache_group, window, sinks, gates):
    w, g = weights(n, D, nh, nkv, hd, F, gates)
    L = LY.FourBitLayer(w, nh, nkv, hd, window=window, sinks=sinks, group=group, residual_scale=0.9)
    cos, sin = tables(512, hd)
    x = torch.randn(2, n, D, device="cuda", generator=g).bfloat16()
    cache = LY.KvCache4(2, 400, nkv, hd, cache_group, x.dtype)
    got = L.forward(x.clone(), cache, cos, sin)
    assert bd.device_status() == 0 and cache.filled == [n, n] and cache.lengths.tolist() == [n, n]
    for b in range(2):
        ref = formula(L, w, x[b], cos, sin, {k: w[k][b] for k in ("gate1", "gate2")} if gates else None, cache_group)
        assert far(got[b], ref) < BOUND, far(got[b], ref)


def test_the_layers_quantiser(bd):
    for cols, group in ((264, 32), (512, 64), (1288, 128)):
        w = torch.randn(48, cols, device="cuda").bfloat16()
        x = torch.randn(4, cols, device="cuda").bfloat16()
        y = torch.empty(4, 48, device="cuda", dtype=torch.bfloat16)
        bd.linear_w4_fwd(x, LY.quantise_rows4(w, group), None, y, group=group)
        ref = x.double() @ in_4_bits(w, group).T
        assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-4 * cols ** 0.5).all()


def test_products_of_many_rows_against_those_of_few(bd, monkeypatch):
    """Matrices back in 16 bits, each value rounded once more (2^-9 of it, as the steps between are), against the 4 bits themselves."""
    D, nh, nkv, hd, F, n = 640, 6, 2, 128, 1288, 100
    w, g = weights(5, D, nh, nkv, hd, F, 0)
    L = LY.FourBitLayer(w, nh, nkv, hd, group=32)
    cos, sin = tables(128, hd)
    x = torch.randn(1, n, D, device="cuda", generator=g).bfloat16()
    many = L.forward(x.clone(), LY.KvCache4(1, n, nkv, hd, 64, x.dtype), cos, sin)
    monkeypatch.setattr(LY.FourBitLayer, "MANY", 10 ** 9)
    few = L.forward(x.clone(), LY.KvCache4(1, n, nkv, hd, 64, x.dtype), cos, sin)
    assert not torch.equal(many, few) and far(many, few) < BOUND


def test_chunks_and_single_tokens_continue_a_prompt(bd):
    D, nh, nkv, hd, F, n = 640, 6, 2, 128, 1280, 150
    w, g = weights(3, D, nh, nkv, hd, F, 0)
    L = LY.FourBitLayer(w, nh, nkv, hd, window=48, sinks=3)
    cos, sin = tables(512, hd)
    x = torch.randn(3, n, D, device="cuda", generator=g).bfloat16()
    whole = L.forward(x.clone(), LY.KvCache4(3, n, nkv, hd, 64, x.dtype), cos, sin)
    cache, parts, at = LY.KvCache4(3, 256, nkv, hd, 64, x.dtype), [], 0
    for t in (cache.rows.k_scales, cache.rows.v_scales):
        t.fill_(float("nan"))                # rows that are not filled yet may hold anything
    for step in [70, 1, 1, 30, 1, 2, 5, 1, 39]:
        parts.append(L.forward(x[:, at:at + step].clone(), cache, cos, sin))
        at += step
    assert at == n and bd.device_status() == 0
    assert far(torch.cat(parts, 1), whole) < BOUND             # (other kernels, other rounding; as above)


def test_sequences_of_different_lengths(bd):
    D, nh, nkv, hd, F = 512, 4, 4, 64, 512
    w, g = weights(4, D, nh, nkv, hd, F, 0, gains=False)
    L = LY.FourBitLayer(w, nh, nkv, hd, window=20, sinks=2)
    cos, sin = tables(256, hd)
    x = torch.randn(6, 101, D, device="cuda", generator=g).bfloat16()
    lens = [100, 3, 57, 20, 99, 1]
    cache = LY.KvCache4(6, 128, nkv, hd, 32, x.dtype)
    for b, m in enumerate(lens):                                       # prompts one by one, each into its own rows
        one = LY.KvCache4(1, 128, nkv, hd, 32, x.dtype)
        one.rows = bd.Cache4(*(getattr(cache.rows, s)[b:b + 1] for s in bd.Cache4.__slots__))
        L.forward(x[b:b + 1, :m].clone(), one, cos, sin)
        cache.filled[b] = m
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    last = torch.stack([x[b, m] for b, m in enumerate(lens)])[:, None]
    got = L.forward(last.clone(), cache, cos, sin)
    for b, m in enumerate(lens):
        assert far(got[b, 0], formula(L, w, x[b, :m + 1], cos, sin, None, 32)[m]) < BOUND


def test_refusals(bd):
    w, g = weights(5, 256, 2, 2, 64, 256, 0)
    L = LY.FourBitLayer(w, 2, 2, 64, window=8)
    cos, sin = tables(16, 64)
    cache = LY.KvCache4(1, 12, 2, 64, 64, torch.bfloat16)
    x = torch.randn(1, 13, 256, device="cuda").bfloat16()
    for bad in (x, x.expand(2, 13, 256), x[:, :, :128]):
        with pytest.raises(bd.BdattnError):
            L.forward(bad, cache, cos, sin)
    assert cache.filled == [0] and L.forward(x[:, :0], cache, cos, sin).shape[1] == 0
