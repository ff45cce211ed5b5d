"""One causal pre-norm layer over a stream of tokens: the operators of the text and
prefix layers in front of a denoiser, put together as such a layer uses them.

    rows of 8 bits   <- add_rmsnorm_fwd (the stream, or the stream + the last branch)
    Q, K, V          <- linear_act_fwd  (8-bit rows and weights)
    Q, K             <- rmsnorm_rope    (per-head norm where gains are given, RoPE; K into the cache)
    attention        <- sdpa_window_fwd (sliding window, sinks, grouped heads, lengths on the device)
    branch           <- linear_act_fwd  (16-bit output projection)
    stream, rows     <- add_rmsnorm_fwd (the branch added, the stream updated in place, 8 bits)
    hidden           <- linear_act_fwd  (8-bit rows and weights, activation)
    stream           <- linear_act_fwd  (16-bit down projection, the residual in its epilogue)

A call takes any number of new tokens of every sequence: a whole prompt, a chunk of it, one
token.  Torch provides memory, the copy of V's new rows into the cache (one a sequence) and the addition to the lengths; nothing
is kept between calls but the weights and the cache.  Where the new rows go and the RoPE positions are numbers of the host, so a
captured call would write the same rows again: of the calls above only the attention follows lengths on the device.
"""
from __future__ import annotations

import brodiffusion_b200 as bd

E4M3_MAX = 448.0


def quantise_rows(w):
    """A matrix in e4m3 and the FP32 scales of its rows (weights, once at load)."""
    import torch
    scale = w.float().abs().amax(1).clamp_min(1e-30) / E4M3_MAX
    return (w.float() / scale[:, None]).to(torch.float8_e4m3fn), scale


class KvCache:
    """K and V rows of ``batch`` sequences, ``lengths`` filled (INT32 on the device, and ``filled`` on the host)."""

    def __init__(self, batch, capacity, num_kv_heads, head_dim, dtype, device="cuda"):
        import torch
        self.k = torch.empty(batch, capacity, num_kv_heads * head_dim, device=device, dtype=dtype)
        self.v = torch.empty_like(self.k)
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)
        self.filled = [0] * batch


class CausalLayer:
    """``weights``: norm1, norm2 (D), wqkv ((nh + 2 nkv) * hd, D), wo (D, nh * hd), w_up (F, D), w_down (D, F), and
    optionally q_gain, k_gain (hd), b_up (F), b_down (D), all of one 16-bit dtype.  ``cos`` / ``sin``: FP32 RoPE
    tables (positions, hd / 2), such as ``rope_tables_qwen`` gives for text."""

    def __init__(self, weights, num_heads, num_kv_heads, head_dim, *, window, sinks=0, act="gelu_tanh", eps=1e-6):
        self.w = dict(weights)
        self.nh, self.nkv, self.hd = num_heads, num_kv_heads, head_dim
        self.window, self.sinks, self.act, self.eps = window, sinks, act, eps
        self.wqkv, self.wqkv_scale = quantise_rows(weights["wqkv"])
        self.w_up, self.w_up_scale = quantise_rows(weights["w_up"])

    def _rows8(self, x, gain, **kw):
        import torch
        out = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
        scale = torch.empty(x.shape[0], device=x.device, dtype=torch.float32)
        bd.add_rmsnorm_fwd(x, out, gain, out_scale=scale, eps=self.eps, **kw)
        return out, scale

    def forward(self, stream, cache, cos, sin):
        """``stream`` (B, L, D): the hidden states of L new tokens of every sequence, updated in place.  Their K and V go
        behind the cache's rows.  A call that raises leaves the cache's lengths as they were (the stream may be half updated)."""
        import torch
        B, L, D = stream.shape
        w, nh, nkv, hd = self.w, self.nh, self.nkv, self.hd
        if B != cache.k.shape[0] or not stream.is_contiguous():
            raise bd.BdattnError("stream must be dense, with a sequence for every one of the cache")
        if L == 0:
            return stream
        if max(cache.filled) + L > min(cache.k.shape[1], cos.shape[0]):
            raise bd.BdattnError(f"{L} new tokens do not fit the cache or the RoPE tables")
        rows = stream.view(B * L, D)
        new = lambda *shape: torch.empty(*shape, device=stream.device, dtype=stream.dtype)

        x8, xs = self._rows8(rows, w["norm1"])
        qkv = new(B, L, (nh + 2 * nkv) * hd)
        bd.linear_act_fwd(x8, self.wqkv, None, qkv.view(B * L, -1), x_scale=xs, w_scale=self.wqkv_scale)
        q, k, v = qkv.split([nh * hd, nkv * hd, nkv * hd], 2)
        for b0 in range(0, B, 4):            # four jobs to a launch
            job = lambda x, out, gain, b: dict(x=x[b], out=out, gain=w.get(gain), cos=cos, sin=sin, rope_row0=cache.filled[b])
            group = range(b0, min(b0 + 4, B))
            bd.rmsnorm_rope([job(q, q[b], "q_gain", b) for b in group], nh, hd, eps=self.eps)
            bd.rmsnorm_rope([job(k, cache.k[b, cache.filled[b]:cache.filled[b] + L], "k_gain", b) for b in group], nkv, hd, eps=self.eps)
        for b in range(B):
            cache.v[b, cache.filled[b]:cache.filled[b] + L].copy_(v[b])
        cache.lengths += L
        try:
            self._behind_the_cache(rows, q, cache, max(cache.filled) + L)
        except BaseException:
            cache.lengths -= L               # the rows behind the lengths are nobody's
            raise
        cache.filled[:] = [n + L for n in cache.filled]
        return stream

    def _behind_the_cache(self, rows, q, cache, most):
        """Attention over the first ``most`` rows of the cache (no row behind the longest sequence is looked at) and what follows."""
        import torch
        w, D = self.w, rows.shape[1]
        new = lambda *shape: torch.empty(*shape, device=rows.device, dtype=rows.dtype)
        att = new(q.shape)
        bd.sdpa_window_fwd(q, cache.k[:, :most], cache.v[:, :most], att, self.nh, window=self.window, sinks=self.sinks,
                           num_kv_heads=self.nkv, kv_len=cache.lengths)
        branch = new(len(rows), D)
        bd.linear_act_fwd(att.view(len(rows), -1), w["wo"], None, branch)

        x8, xs = self._rows8(branch, w["norm2"], residual=rows, residual_out=rows)
        hidden = new(len(rows), w["w_up"].shape[0])
        bd.linear_act_fwd(x8, self.w_up, w.get("b_up"), hidden, act=self.act, x_scale=xs, w_scale=self.w_up_scale)
        bd.linear_act_fwd(hidden, w["w_down"], w.get("b_down"), rows, residual=rows)
