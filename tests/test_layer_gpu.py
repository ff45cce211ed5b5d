"""A causal layer over a stream (brodiffusion_b200/layer.py) against its steps in 64 bits, and its calls against one
another: a prompt at once, in chunks and token by token."""
import math

import pytest
import torch

from brodiffusion_b200 import layer as LY

pytestmark = pytest.mark.gpu


def make(seed, D, nh, nkv, hd, F, dtype=torch.bfloat16, gains=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, scale: (scale * torch.randn(*s, device="cuda", generator=g)).to(dtype)
    w = dict(norm1=1 + r(D, scale=0.02), norm2=1 + r(D, scale=0.02), wqkv=r((nh + 2 * nkv) * hd, D, scale=D ** -0.5),
             wo=r(D, nh * hd, scale=(nh * hd) ** -0.5), w_up=r(F, D, scale=D ** -0.5), w_down=r(D, F, scale=F ** -0.5),
             b_up=r(F, scale=0.02), b_down=r(D, scale=0.02))
    if gains:
        w.update(q_gain=1 + r(hd, scale=0.02), k_gain=1 + r(hd, scale=0.02))
    return w, g


def tables(n, hd):
    f = 10000.0 ** (-torch.arange(0, hd, 2, device="cuda").double() / hd)
    a = torch.arange(n, device="cuda").double()[:, None] * f
    return a.cos().float(), a.sin().float()


def round8(y):
    s = y.abs().amax(1, keepdim=True) / 448
    return (y / s).float().to(torch.float8_e4m3fn).double() * s


def rms(x, gain, eps=1e-6):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if gain is None else y * gain.double()


def rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def formula(L, stream, cos, sin):
    """One sequence from its start, all steps in 64 bits; 8-bit operands rounded as the layer holds them."""
    w, nh, nkv, hd = L.w, L.nh, L.nkv, L.hd
    n = stream.shape[0]
    wqkv = L.wqkv.double() * L.wqkv_scale.double()[:, None]
    w_up = L.w_up.double() * L.w_up_scale.double()[:, None]
    x = stream.double()
    q, k, v = (round8(rms(x, w["norm1"])) @ wqkv.T).split([nh * hd, nkv * hd, nkv * hd], 1)
    q, k, v = (t.view(n, -1, hd) for t in (q, k, v))
    q = rotate(rms(q, w.get("q_gain")) if "q_gain" in w else q, cos[:n], sin[:n])
    k = rotate(rms(k, w.get("k_gain")) if "k_gain" in w else k, cos[:n], sin[:n])
    k, v = (t.repeat_interleave(nh // nkv, 1) for t in (k, v))
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    seen = (j <= i) & ((i - j < L.window) | (j < L.sinks)) if L.window else j <= i
    s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd)
    att = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, -math.inf), -1), v).reshape(n, -1)
    x = x + att @ w["wo"].double().T
    h = round8(rms(x, w["norm2"])) @ w_up.T + w["b_up"].double()
    h = torch.nn.functional.gelu(h, approximate="tanh")
    return x + h @ w["w_down"].double().T + w["b_down"].double()


def far(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("D,nh,nkv,hd,F,n", [(512, 4, 2, 64, 1024, 200), (640, 6, 2, 128, 1280, 333), (1280, 8, 8, 64, 2560, 40)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 4)])
def test_a_prompt_against_the_formulas(bd, D, nh, nkv, hd, F, n, window, sinks):
    w, g = make(n, D, nh, nkv, hd, F)
    L = LY.CausalLayer(w, nh, nkv, hd, window=window, sinks=sinks)
    cos, sin = tables(512, hd)
    x = torch.randn(2, n, D, device="cuda", generator=g).bfloat16()
    cache = LY.KvCache(2, 400, nkv, hd, x.dtype)
    got = L.forward(x.clone(), cache, cos, sin)
    assert bd.device_status() == 0 and cache.filled == [n, n] and cache.lengths.tolist() == [n, n]
    for b in range(2):
        ref = formula(L, x[b], cos, sin)
        # Rounding of the 16-bit tensors between the steps, 2^-9 rms of each: six of them in a row of the branches, and
        # 8-bit values that a 16-bit rounding ahead of them moved over a step's middle (2^-9 / 2^-4 of them, by 2^-4 each: 2^-6.5 ...
        # of the value, 0.011, at most): below 0.02 of the branches, which are below the stream that they are added to
        assert far(got[b], ref) < 0.02


def test_chunks_and_single_tokens_continue_a_prompt(bd):
    D, nh, nkv, hd, F, n = 640, 6, 2, 128, 1280, 150
    w, g = make(3, D, nh, nkv, hd, F)
    L = LY.CausalLayer(w, nh, nkv, hd, window=48, sinks=3)
    cos, sin = tables(512, hd)
    x = torch.randn(3, n, D, device="cuda", generator=g).bfloat16()
    whole = L.forward(x.clone(), LY.KvCache(3, n, nkv, hd, x.dtype), cos, sin)
    cache, parts, at = LY.KvCache(3, 256, nkv, hd, x.dtype), [], 0
    cache.k.fill_(float("nan")), cache.v.fill_(float("nan"))          # rows that are not filled yet may hold anything
    for step in [70, 1, 1, 30, 1, 2, 5, 1, 39]:
        parts.append(L.forward(x[:, at:at + step].clone(), cache, cos, sin))
        at += step
    assert at == n and bd.device_status() == 0
    assert far(torch.cat(parts, 1), whole) < 0.02          # (other kernels, other rounding; as above)


def test_sequences_of_different_lengths(bd):
    D, nh, nkv, hd, F = 512, 4, 4, 64, 512
    w, g = make(4, D, nh, nkv, hd, F, gains=False)
    L = LY.CausalLayer(w, nh, nkv, hd, window=20, sinks=2, act="gelu_tanh")
    cos, sin = tables(256, hd)
    cache = LY.KvCache(6, 128, nkv, hd, torch.bfloat16)
    x = torch.randn(6, 101, D, device="cuda", generator=g).bfloat16()
    lens = [100, 3, 57, 20, 99, 1]
    for b, m in enumerate(lens):                                       # prompts one by one, each into its own rows
        one = LY.KvCache(1, 128, nkv, hd, x.dtype)
        one.k, one.v = cache.k[b:b + 1], cache.v[b:b + 1]
        L.forward(x[b:b + 1, :m].clone(), one, cos, sin)
        cache.filled[b] = m
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    last = torch.stack([x[b, m] for b, m in enumerate(lens)])[:, None]
    got = L.forward(last.clone(), cache, cos, sin)
    for b, m in enumerate(lens):
        assert far(got[b, 0], formula(L, x[b, :m + 1], cos, sin)[m]) < 0.02


def test_refusals(bd):
    w, g = make(5, 256, 2, 2, 64, 256)
    L = LY.CausalLayer(w, 2, 2, 64, window=8)
    cos, sin = tables(16, 64)
    cache = LY.KvCache(1, 12, 2, 64, torch.bfloat16)
    x = torch.randn(1, 13, 256, device="cuda").bfloat16()
    for bad in (x, x.expand(2, 13, 256), x[:, :, :128]):
        with pytest.raises(bd.BdattnError):
            L.forward(bad, cache, cos, sin)
    assert cache.filled == [0] and L.forward(x[:, :0], cache, cos, sin).shape[1] == 0
