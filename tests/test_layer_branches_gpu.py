"""What a causal layer adds to its stream, a branch at a time, against its steps in 64 bits, by the size of the branch itself:
the stream is a hundredth of the usual one (the norm takes that out), so that it does not hide what is added to it.  The
formula runs on the CPU, and with a mistake planted in it the layer has to be far from it."""
import math

import pytest
import torch

import test_layer_gpu as T
from brodiffusion_b200 import layer as LY

pytestmark = pytest.mark.gpu


def formula(L, stream, cos, sin, window, sinks, act):
    """One sequence from its start: (attention branch, feed-forward branch), all steps in 64 bits but for the 8-bit rows."""
    w = {n: t.cpu().double() for n, t in L.w.items()}
    nh, nkv, hd, n = L.nh, L.nkv, L.hd, stream.shape[0]
    wqkv, w_up = ((a.cpu().double() * s.cpu().double()[:, None]) for a, s in ((L.wqkv, L.wqkv_scale), (L.w_up, L.w_up_scale)))
    x, cos, sin = stream.cpu().double(), cos[:n].cpu(), sin[:n].cpu()
    q, k, v = (T.round8(T.rms(x, w["norm1"])) @ wqkv.T).split([nh * hd, nkv * hd, nkv * hd], 1)
    q, k, v = (t.view(n, -1, hd) for t in (q, k, v))
    q, k = (T.rotate(T.rms(t, w[g]), cos, sin) for t, g in ((q, "q_gain"), (k, "k_gain")))
    k, v = (t.repeat_interleave(nh // nkv, 1) for t in (k, v))
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd)
    att = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, -math.inf), -1), v).reshape(n, -1) @ w["wo"].T
    h = T.round8(T.rms(x + att, w["norm2"])) @ w_up.T + w["b_up"]
    h = torch.nn.functional.silu(h) if act == "silu" else torch.nn.functional.gelu(h, approximate="tanh")
    return att, h @ w["w_down"].T + w["b_down"]


def added(bd, w, n, window, sinks, seed):
    nh, nkv, hd, D = 4, 2, 64, 512
    L = LY.CausalLayer(w, nh, nkv, hd, window=window, sinks=sinks)
    cos, sin = T.tables(512, hd)
    x = (0.01 * torch.randn(2, n, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))).bfloat16()
    got = L.forward(x.clone(), LY.KvCache(2, n, nkv, hd, x.dtype), cos, sin)
    assert bd.device_status() == 0
    return L, x, (got.double() - x.double()).cpu(), cos, sin


@pytest.mark.parametrize("n", [70, 200, 333])
@pytest.mark.parametrize("window,sinks", [(64, 4), (33, 0)])
def test_the_attention_branch(bd, n, window, sinks):
    w, _ = T.make(n, 512, 4, 2, 64, 1024)
    w["w_down"], w["b_down"] = torch.zeros_like(w["w_down"]), torch.zeros_like(w["b_down"])
    L, x, got, cos, sin = added(bd, w, n, window, sinks, n)
    for b in range(2):
        f = lambda window, sinks: formula(L, x[b], cos, sin, window, sinks, "gelu_tanh")[0]
        # Roundings to BF16, 2^-8 / sqrt(3) / 1.4 = 0.0016 rms of each: Q, K, V, their norm and RoPE, the weights, the heads'
        # outputs, the branch, the stream.  Four of them are in a score, 0.0033 of a weight; six on the way of V, 0.004; values of
        # 8 bits that an FP32 rounding moved over a step's middle (1e-5 / 2^-4 of them, by 2^-3) 0.0016: together 0.0055, twice that.
        assert T.far(got[b], f(window, sinks)) < 0.011
        # one key of `window` less or more, a sink less: sqrt(1 / window) of the rows that have as many keys, 0.12 and more
        past = slice(window + 8, n)
        if n > window + 8:
            for wrong in (f(window - 1, sinks), f(window + 1, sinks), f(window, sinks - 1 if sinks else 1)):
                assert T.far(got[b][past], wrong[past]) > 0.022


@pytest.mark.parametrize("n", [1, 40, 200])
def test_the_feed_forward_branch(bd, n):
    w, _ = T.make(n, 512, 4, 2, 64, 1024)
    w["wo"] = torch.zeros_like(w["wo"])
    L, x, got, cos, sin = added(bd, w, n, 64, 4, n)
    for b in range(2):
        f = lambda act: formula(L, x[b], cos, sin, 64, 4, act)[1]
        # hidden, output: 0.0016 rms each, 8-bit values as above 0.0016: 0.0028, twice that
        assert T.far(got[b], f("gelu_tanh")) < 0.0056
        assert T.far(got[b], f("silu")) > 0.05
