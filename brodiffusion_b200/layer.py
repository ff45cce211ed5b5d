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

``FourBitLayer`` is such a layer with a norm on both sides of each block, served with weights and cache in 4 bits:

    rows             <- add_rmsnorm_fwd   (16 bits, the stream's first norm)
    Q, K, V          <- linear_w4_fwd     (a few rows), or w4_unpack and linear_act_fwd (many); so all products
    Q, K             <- rmsnorm_rope
    cache            <- cache4_append     (to the places that the lengths on the device say)
    attention        <- sdpa_cache4_fwd   (a few new tokens), or cache4_read and sdpa_window_fwd (a prompt)
    branch           <- linear_w4_fwd
    stream, rows     <- sandwich_norm_fwd (the branch's norm and gate, the stream's scale, the next block's norm)
    hidden, branch   <- linear_w4_fwd     (activation; down projection)
    stream           <- sandwich_norm_fwd
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


def quantise_rows4(w, group):
    """A matrix in 4-bit groups of its rows, packed for ``linear_w4_fwd`` (weights, once at load)."""
    import torch
    rows, cols = w.shape
    whole = -(-cols // group) * group
    if whole > cols:                         # a short last group is one of the columns that there are
        w = torch.cat([w, w[:, -1:].expand(rows, whole - cols)], 1)
    g = w.float().view(rows, -1, group)
    low, top = g.amin(2), g.amax(2)
    step = ((top - low) / 15).to(w.dtype)
    s = step.float()[:, :, None]
    codes = torch.where(s > 0, ((g - low[:, :, None]) / torch.where(s > 0, s, 1)).round().clamp(0, 15), 0)
    codes = codes.to(torch.uint8).view(rows, whole)[:, :cols]
    packed = torch.empty(bd.w4_bytes(rows, cols, group), device=w.device, dtype=torch.uint8)
    bd.w4_pack((codes[:, 0::2] | codes[:, 1::2] << 4).contiguous(), torch.stack([step, low.to(w.dtype)], 2), packed, group=group)
    return packed


class KvCache4:
    """K and V rows of ``batch`` sequences in 4-bit groups, ``lengths`` filled (INT32 on the device, and ``filled`` on the host)."""

    def __init__(self, batch, capacity, num_kv_heads, head_dim, group, dtype, device="cuda"):
        import torch
        self.rows = bd.Cache4.empty(batch, num_kv_heads, capacity, head_dim, group, dtype, device)
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)
        self.filled = [0] * batch


class FourBitLayer:
    """``weights`` as for ``CausalLayer``, and post1, post2 (D), the gains behind the two blocks; optionally gate1, gate2 (D)
    or (n, D), a vector for each batch / n sequences.  ``group``: columns of W to a step and a low."""

    # The attention reads 16-bit rows, read back from the cache, from PROMPT new tokens of a sequence and 64 rows of heads to a K/V head on: it takes 128 of
    # those at a time, the kernel over 4 bits sixteen.  Heads of 128, groups of 32, 8 K/V heads, us from the 4 bits and by way of 16:
    #   24 heads, 8 tokens over 1000 / 8000 / 32768 keys 12.0, 26.6, 72 and 12.5, 22.7, 75, of 32 sequences of 8192 259 and 448;
    #   32 tokens 15.0, 43, 133 and 14.4, 37, 127, of 32 sequences 722 and 720; 64 tokens 26, 82, 223 and 17, 57, 207, of 32 sequences 1352 and 721;
    #   8 heads, 8 sequences of 8000: 32 tokens 84 and 122, 64 tokens 162 and 157.
    # With a window only what it shows is read back, where all sequences are as long (32 sequences of 8192, window 1024: 16 tokens 88 and 104, 32 tokens
    # 162 and 133, with all rows read back 344).
    PROMPT = 32
    # Rows from which on a matrix goes back to 16 bits ahead of its product, a workspace of the call's, and half as many more for one of less
    # than 2^23 values (us in 4 bits and so, groups of 32: 10240 x 2560, 32 rows 21.2 and 22.3, 48 rows 28 and 23, 1536 rows 606 and 70; 5120 x 5120, 32 rows 20.5 and
    # 24.7, 64 rows 33 and 25; 2560 x 2560, 64 rows 12.1 and 14.2, 96 rows 16.0 and 14.4; 1280 x 1280, 64 rows 5.8 and 8.0, 128 rows 7.8 and 7.6).
    MANY = 64

    def __init__(self, weights, num_heads, num_kv_heads, head_dim, *, window=0, sinks=0, act="gelu_tanh", eps=1e-6, group=64,
                 residual_scale=1.0):
        import torch
        self.w = {n: t for n, t in weights.items() if n not in ("wqkv", "wo", "w_up", "w_down")}
        self.dtype = weights["wqkv"].dtype   # (of the steps and lows, which the packed bytes do not say)
        if self.dtype not in (torch.bfloat16, torch.float16) or any(weights[n].dtype != self.dtype for n in ("wo", "w_up", "w_down")):
            raise bd.BdattnError("wqkv, wo, w_up and w_down must be of one 16-bit dtype")
        self.nh, self.nkv, self.hd = num_heads, num_kv_heads, head_dim
        self.window, self.sinks, self.act, self.eps, self.group, self.scale = window, sinks, act, eps, group, residual_scale
        self.widths = {n: weights[n].shape[0] for n in ("wqkv", "wo", "w_up", "w_down")}
        self.packed = {n: quantise_rows4(weights[n], group) for n in self.widths}

    def _product(self, x, name, bias=None, **kw):
        import torch
        y = torch.empty(len(x), self.widths[name], device=x.device, dtype=x.dtype)
        if len(x) < (self.MANY if self.widths[name] * x.shape[1] >= 1 << 23 else self.MANY * 3 // 2):
            bd.linear_w4_fwd(x, self.packed[name], bias, y, group=self.group, **kw)
        else:
            w = torch.empty(self.widths[name], x.shape[1], device=x.device, dtype=x.dtype)
            bd.w4_unpack(self.packed[name], w, group=self.group)
            bd.linear_act_fwd(x, w, bias, y, **kw)
        return y

    def forward(self, stream, cache, cos, sin):
        """``stream`` (B, L, D): the hidden states of L new tokens of every sequence, updated in place; their K and V go behind the
        cache's rows.  A call that raises leaves the cache's lengths as they were (the stream may be half updated)."""
        import torch
        B, L, D = stream.shape
        w, nh, nkv, hd = self.w, self.nh, self.nkv, self.hd
        if B != len(cache.filled) or not stream.is_contiguous():
            raise bd.BdattnError("stream must be dense, with a sequence for every one of the cache")
        if stream.dtype != self.dtype:
            raise bd.BdattnError(f"stream must have the weights' dtype ({self.dtype}, got {stream.dtype})")
        if L == 0:
            return stream
        if max(cache.filled) + L > min(cache.rows.rows, cos.shape[0]):
            raise bd.BdattnError(f"{L} new tokens do not fit the cache or the RoPE tables")
        for name in ("gate1", "gate2"):
            if name in w and w[name].dim() == 2 and (len(w[name]) < 1 or B % len(w[name])):
                raise bd.BdattnError(f"{name} must have a vector for each batch / n sequences ({len(w[name])} for {B})")
        rows = stream.view(B * L, D)
        x = torch.empty_like(rows)
        bd.add_rmsnorm_fwd(rows, x, w["norm1"], eps=self.eps)
        q, k, v = self._product(x, "wqkv").view(B, L, -1).split([nh * hd, nkv * hd, nkv * hd], 2)
        for b0 in range(0, B, 4):            # four jobs to a launch
            job = lambda t, gain, b: dict(x=t[b], out=t[b], gain=w.get(gain), cos=cos, sin=sin, rope_row0=cache.filled[b])
            group = range(b0, min(b0 + 4, B))
            bd.rmsnorm_rope([job(q, "q_gain", b) for b in group], nh, hd, eps=self.eps)
            bd.rmsnorm_rope([job(k, "k_gain", b) for b in group], nkv, hd, eps=self.eps)
        cache.lengths += L
        try:
            bd.cache4_append(k, v, cache.rows, kv_len=cache.lengths)
            self._behind_the_cache(rows, x, q, cache, min(cache.filled) + L, max(cache.filled) + L)
        except BaseException:
            cache.lengths -= L               # the rows behind the lengths are nobody's
            raise
        cache.filled[:] = [n + L for n in cache.filled]
        return stream

    def _behind_the_cache(self, rows, x, q, cache, least, most):
        """Attention over the first ``most`` rows of the cache (no row behind the longest sequence is looked at; the shortest has ``least``) and
        what follows."""
        import torch
        w, held = self.w, cache.rows.first(most)
        att = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        seen = dict(window=self.window, sinks=self.sinks, kv_len=cache.lengths)
        new = q.shape[1]
        if new < self.PROMPT or new * self.nh < 64 * self.nkv:
            bd.sdpa_cache4_fwd(q, held, att, self.nh, **seen)
        else:
            tail, first, places = self.window + new - 1, 0, {}
            if 0 < self.window and self.sinks + tail <= least:           # the first rows that stay visible, and the last that any new token sees
                first, most, places = self.sinks, self.sinks + tail, dict(kv_len=seen.pop("kv_len"))
            k, v = (torch.empty(q.shape[0], most, self.nkv * self.hd, device=q.device, dtype=q.dtype) for _ in range(2))
            if first > 0:
                bd.cache4_read(held.first(first), k[:, :first], v[:, :first])
            bd.cache4_read(held, k[:, first:], v[:, first:], **places)
            bd.sdpa_window_fwd(q, k, v, att, self.nh, num_kv_heads=self.nkv, **seen)
        behind = dict(residual_scale=self.scale, eps=self.eps)
        branch = self._product(att.view(len(rows), -1), "wo")
        bd.sandwich_norm_fwd(branch, rows, rows, w["post1"], gate=w.get("gate1"), gain=w["norm2"], out=x, **behind)
        hidden = self._product(x, "w_up", w.get("b_up"), act=self.act)
        branch = self._product(hidden, "w_down", w.get("b_down"))
        bd.sandwich_norm_fwd(branch, rows, rows, w["post2"], gate=w.get("gate2"), **behind)
