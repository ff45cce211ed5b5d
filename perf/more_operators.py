"""The operators of a causal layer whose weights and cache are held in 4 bits, as timed cases.

    norm     the branch's own norm, its gate and the stream's scale, the addition to the
             stream and the norm in front of the next block, to 16 bits or to e4m3
    linear   X W^T for a few rows, W in 4-bit codes with a step and a lowest value per
             group of columns; bias, activation, gate and residual behind it
    append   new rows of K and V into a cache of such codes, and the same rows read back
    cache    causal attention over that cache with a sliding window and first keys that
             stay visible: single tokens, drafted ones, a chunk of new rows

A group of values x is held as low = min x, step = (max x - min x) / 15 rounded to the
tensors' type, and codes round((x - low) / step) in 0..15.  Activations are N(0, 1),
weights N(0, 0.02), gains 1 + N(0, 0.02), as everywhere in this repository's tests and
benchmark; channels of K have means of their own.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}
_E4M3_MAX = 448.0
_EPS = 1e-6


def listed():
    return [
        # One new token between two blocks: a single row, 8-bit output for the projection behind it: latency.
        {"name": "norm_one_token", "op": "norm", "rows": 1, "cols": 2560, "gates": 1, "scale": 1.0, "out": "fp8", "dtype": "bf16"},
        # Two images' tokens with a gate vector each, 16-bit output (the rows of a portrait image, 2240 columns).
        {"name": "norm_modulated", "op": "norm", "rows": 4332, "cols": 2240, "gates": 2, "scale": 0.5, "out": "same",
         "dtype": "fp16"},
        # A long prompt, ungated, 8-bit output: bound by memory.
        {"name": "norm_long", "op": "norm", "rows": 16384, "cols": 5120, "gates": 0, "scale": 1.0, "out": "fp8", "dtype": "bf16"},
        # One token through an up projection with activation: the weights' bytes are the time.
        {"name": "linear_one_token", "op": "linear", "rows": 1, "inputs": 2560, "outputs": 10240, "group": 128, "act": "silu",
         "bias": False, "gate": False, "residual": False, "dtype": "bf16"},
        # Eight sequences' single tokens, the finest groups.
        {"name": "linear_tokens", "op": "linear", "rows": 8, "inputs": 5120, "outputs": 5120, "group": 32, "act": "none",
         "bias": True, "gate": False, "residual": True, "dtype": "fp16"},
        # Drafted tokens of a batch, sizes that no tile divides, the last group not whole.
        {"name": "linear_ragged", "op": "linear", "rows": 13, "inputs": 1368, "outputs": 1291, "group": 32, "act": "gelu",
         "bias": True, "gate": False, "residual": True, "dtype": "bf16"},
        # A serving batch of single tokens through a down projection, gated into the stream.
        {"name": "linear_batch", "op": "linear", "rows": 48, "inputs": 10240, "outputs": 2560, "group": 64, "act": "none",
         "bias": True, "gate": True, "residual": True, "dtype": "bf16"},
        # A serving batch's new rows behind caches of different lengths: latency.
        {"name": "append_tokens", "op": "append", "batch": 32, "new": 1, "rows": 4096, "kv_heads": 8, "head_dim": 64, "group": 64,
         "ragged": True, "dtype": "fp16"},
        # Two prompts into their caches, the finest groups: bound by memory.
        {"name": "append_prompts", "op": "append", "batch": 2, "new": 8191, "rows": 16384, "kv_heads": 8, "head_dim": 128,
         "group": 32, "ragged": True, "dtype": "bf16"},
        # One sequence, one token, a short cache: latency.
        {"name": "cache_one_token", "op": "cache", "batch": 1, "new": 1, "rows": 777, "heads": 24, "kv_heads": 8, "head_dim": 128,
         "group": 128, "window": 0, "sinks": 0, "ragged": False, "padded": 0, "dtype": "bf16"},
        # A serving batch of single tokens over long caches of different lengths: the visible rows' bytes are the time.
        {"name": "cache_tokens_ragged", "op": "cache", "batch": 32, "new": 1, "rows": 32768, "heads": 24, "kv_heads": 8,
         "head_dim": 128, "group": 32, "window": 0, "sinks": 0, "ragged": True, "padded": 0, "dtype": "bf16"},
        # A chunk of a left-padded prompt behind what is cached, heads of 64, window and sinks: arithmetic.
        {"name": "cache_chunk", "op": "cache", "batch": 2, "new": 509, "rows": 8009, "heads": 16, "kv_heads": 4, "head_dim": 64,
         "group": 64, "window": 4096, "sinks": 70, "ragged": True, "padded": 37, "dtype": "fp16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "append", "cache"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "norm":
        cols = _log_int(rng, 64, 8192)
        if rng.random() < 0.75:
            cols = (cols + 7) // 8 * 8
        gates = rng.choice([0, 1, _log_int(rng, 2, 8)])
        rows = _log_int(rng, 1, max(2, min(16384, 14336 * 5120 // cols) // max(1, gates))) * max(1, gates)
        return {"op": op, "rows": rows, "cols": cols, "gates": gates, "scale": rng.choice([1.0, 0.5, rng.uniform(0.1, 2.0)]),
                "out": rng.choice(["same", "fp8", "none"]), "dtype": dtype}
    if op == "linear":
        inputs, outputs = 8 * _log_int(rng, 8, 1280), _log_int(rng, 16, 10240)
        if rng.random() < 0.7:
            outputs = (outputs + 7) // 8 * 8
        return {"op": op, "rows": rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 64)]), "inputs": inputs, "outputs": outputs,
                "group": rng.choice([32, 64, 128]), "act": rng.choice(["none", "none", "gelu", "gelu_tanh", "silu"]),
                "bias": rng.random() < 0.6, "gate": rng.random() < 0.3, "residual": rng.random() < 0.5, "dtype": dtype}
    kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= head_dim])
    if op == "append":
        rows = _log_int(rng, 16, 32768)
        batch = _log_int(rng, 1, max(1, min(32, 32768 // rows)))
        return {"op": op, "batch": batch, "new": rng.choice([1, _log_int(rng, 1, min(rows, 16384 // batch))]), "rows": rows,
                "kv_heads": kv_heads, "head_dim": head_dim, "group": group, "ragged": rng.random() < 0.7, "dtype": dtype}
    share = rng.choice([1, 1, 2, 3, 4, 8])
    window, sinks = rng.choice([0, _log_int(rng, 16, 4096)]), rng.choice([0, 4, _log_int(rng, 1, 256)])
    few = rng.random() < 0.7                               # a few new tokens of several sequences, or a chunk of new rows
    batch = _log_int(rng, 1, 32) if few else rng.choice([1, 1, 2])
    new = rng.choice([1, 1, 1, rng.randint(2, 8)]) if few else _log_int(rng, 9, 512)
    most = int(1.6e10 / (4 * batch * new * share * kv_heads * head_dim))       # keys, so that none is dearer than the listed chunk
    rows = new + _log_int(rng, 1 if not few else 8, max(8, min(32768 if few else 16384 // batch, most) - new))
    return {"op": op, "batch": batch, "new": new, "rows": rows, "heads": share * kv_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "group": group, "window": window, "sinks": sinks, "ragged": rng.random() < 0.6,
            "padded": rng.choice([0, 0, rng.randint(1, 40)]), "dtype": dtype}


# --------------------------------------------------- values in 4 bits
def _quantised(x, group):
    """Codes 0..15 (uint8) of the last dimension's groups, and their (step, low) pairs in the type of x."""
    g = x.reshape(*x.shape[:-1], -1, group).float()
    low, top = g.amin(-1), g.amax(-1)
    step = ((top - low) / 15).to(x.dtype)
    s = step.float()[..., None]
    codes = torch.where(s > 0, ((g - low[..., None]) / torch.where(s > 0, s, 1)).round().clamp(0, 15), 0)
    return codes.to(torch.uint8).reshape(x.shape), torch.stack([step, low.to(x.dtype)], -1)


def _pairs(codes):
    """Two codes to a byte, that of the even column in its low half."""
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _values(pairs, scales, group):
    """What packed codes stand for: low + step * code."""
    codes = torch.stack([pairs & 15, pairs >> 4], -1).flatten(-2).float()
    s = scales.float()
    if codes.shape[-1] % group:                            # the last group is not whole
        s = s.repeat_interleave(group, -2)[..., :codes.shape[-1], :]
        return s[..., 1] + s[..., 0] * codes
    return (s[..., 1:] + s[..., :1] * codes.unflatten(-1, (-1, group))).flatten(-2)


class _Make:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def act(self, dtype, *shape):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=self.gen)


def _lengths(case):
    """Filled rows of each sequence's cache."""
    rows, new = case["rows"], case["new"]
    if not case["ragged"]:
        return [rows] * case["batch"]
    return [max(new, rows - (b * 2654435761 % 4096) * (rows - rows // 3) // 4096) for b in range(case["batch"])]


def _inputs(case, seed):
    """The call's operands in plain tensors."""
    m, dtype = _Make(seed), _DTYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s = {"x": m.act(dtype, rows, cols), "residual": m.act(dtype, rows, cols), "post": 1 + 0.02 * m.act(dtype, cols),
             "gain": 1 + 0.02 * m.act(dtype, cols), "gate": None}
        if case["gates"]:
            s["gate"] = 0.5 * m.act(dtype, case["gates"], cols)
        return s
    if case["op"] == "linear":
        rows, inputs, outputs, group = case["rows"], case["inputs"], case["outputs"], case["group"]
        whole = -(-inputs // group) * group
        w = 0.02 * m.act(dtype, outputs, whole)
        if whole > inputs:                                 # the last group is one of the columns that there are
            w[:, inputs:] = w[:, inputs - 1:inputs]
        codes, scales = _quantised(w, group)
        s = {"x": m.act(dtype, rows, inputs), "codes": _pairs(codes[:, :inputs].contiguous()), "scales": scales, "bias": None,
             "gate": None, "residual": None}
        if case["bias"]:
            s["bias"] = 0.02 * m.act(dtype, outputs)
        if case["gate"]:
            s["gate"] = 0.5 * m.act(dtype, outputs)
        if case["residual"]:
            s["residual"] = m.act(dtype, rows, outputs)
        return s
    b, nkv, hd, rows = case["batch"], case["kv_heads"], case["head_dim"], case["rows"]
    kv_len = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32) if case["ragged"] else None
    means = m.act(dtype, nkv * hd)
    if case["op"] == "append":
        return {"k": m.act(dtype, b, case["new"], nkv * hd) + means, "v": m.act(dtype, b, case["new"], nkv * hd), "kv_len": kv_len}
    s = {"q": m.act(dtype, b, case["new"], case["heads"] * hd), "k": m.act(dtype, b, rows, nkv * hd).add_(means),
         "v": m.act(dtype, b, rows, nkv * hd), "kv_len": kv_len, "key_mask": None}
    if case["padded"]:
        s["key_mask"] = (torch.arange(rows, device="cuda") >= case["padded"]).float()
    return s


def _by_heads(x, heads):
    """(B, rows, heads * hd) -> (B, heads, rows, hd)"""
    return x.view(*x.shape[:2], heads, -1).transpose(1, 2)


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    dtype = _DTYPES[case["dtype"]]
    if own:
        import brodiffusion_b200 as bd
    if case["op"] == "norm":
        s["residual_out"], s["out"], s["out_scale"] = torch.empty_like(s["x"]), None, None
        if case["out"] == "same":
            s["out"] = torch.empty_like(s["x"])
        if case["out"] == "fp8":
            s["out"] = torch.empty(s["x"].shape, device="cuda", dtype=torch.float8_e4m3fn)
            s["out_scale"] = torch.empty(case["rows"], device="cuda")
    elif case["op"] == "linear":
        s["y"] = torch.empty(case["rows"], case["outputs"], device="cuda", dtype=dtype)
        if own:
            s["w"] = torch.empty(bd.w4_bytes(case["outputs"], case["inputs"], case["group"]), device="cuda", dtype=torch.uint8)
            bd.w4_pack(s.pop("codes"), s.pop("scales"), s["w"], group=case["group"])
    elif case["op"] == "append":
        s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        if own:
            s["cache"] = bd.Cache4.empty(case["batch"], case["kv_heads"], case["rows"], case["head_dim"], case["group"], dtype)
    else:
        s["out"] = torch.empty_like(s["q"])
        k, v = s.pop("k"), s.pop("v")
        if own:
            s["cache"] = bd.Cache4.empty(case["batch"], case["kv_heads"], case["rows"], case["head_dim"], case["group"], dtype)
            bd.cache4_append(k, v, s["cache"])
        else:
            for name, x in (("k", k), ("v", v)):           # an item at a time: the FP32 steps are large
                parts = [_quantised(_by_heads(x[b:b + 1], case["kv_heads"]), case["group"]) for b in range(case["batch"])]
                s[name + "_codes"] = torch.cat([_pairs(c) for c, _ in parts])
                s[name + "_scales"] = torch.cat([p for _, p in parts])
    return s


# ------------------------------------------------------------- plain forms
def _plain_norm(s):
    c = s["case"]
    x, r = s["x"].float(), s["residual"].float()
    branch = x * torch.rsqrt((x * x).mean(1, keepdim=True) + _EPS) * s["post"].float()
    if s["gate"] is not None:
        branch = (branch.view(c["gates"], -1, c["cols"]) * s["gate"].float()[:, None]).view(x.shape)
    h = c["scale"] * r + branch
    out = {"residual_out": h.to(s["x"].dtype)}
    if c["out"] == "none":
        return out
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS) * s["gain"].float()
    if c["out"] == "same":
        return {**out, "out": y.to(s["x"].dtype)}
    scale = y.abs().amax(1) * (1 / _E4M3_MAX)
    q = y / torch.where(scale > 0, scale, 1)[:, None]
    return {**out, "out": q.clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn), "scale": scale}


def _plain_act(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _plain_linear(s):
    z = s["x"].float() @ _values(s["codes"], s["scales"], s["case"]["group"]).t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _plain_act(z, s["case"]["act"])
    if s["gate"] is not None:
        y = y * s["gate"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["y"].dtype)


def _plain_append(s):
    """What the cache holds for the new rows."""
    c, out = s["case"], []
    for x in (s["k"], s["v"]):
        codes, scales = _quantised(_by_heads(x, c["kv_heads"]), c["group"])
        held = _values(_pairs(codes), scales, c["group"])
        out.append(held.transpose(1, 2).reshape(x.shape).to(x.dtype))
    return out


def _plain_cache(s):
    c = s["case"]
    b, new, rows, nkv, hd = c["batch"], c["new"], c["rows"], c["kv_heads"], c["head_dim"]
    k, v = (_values(s[n + "_codes"], s[n + "_scales"], c["group"]) for n in ("k", "v"))
    q = s["q"].float().view(b, new, nkv, c["heads"] // nkv, hd).permute(0, 2, 3, 1, 4).reshape(b, nkv, -1, hd)
    key = torch.arange(rows, device="cuda")
    length = s["kv_len"].long() if s["kv_len"] is not None else torch.full((b,), rows, device="cuda")
    pos = (length - new)[:, None] + torch.arange(new, device="cuda")
    seen = key <= pos[:, :, None]
    if c["window"]:
        seen = seen & ((key > pos[:, :, None] - c["window"]) | (key < c["sinks"]))
    if s["key_mask"] is not None:
        seen = seen & (s["key_mask"] != 0)
    score = (q @ k.transpose(2, 3) * (1 / math.sqrt(hd))).view(b, nkv, -1, new, rows)
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, 1)).view(b, nkv, -1, rows)
    o = (p @ v).view(b, nkv, -1, new, hd).permute(0, 3, 1, 2, 4)
    return o.reshape(s["q"].shape).to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "append": _plain_append, "cache": _plain_cache}[c["op"]](s)
    import brodiffusion_b200 as bd
    if c["op"] == "norm":
        bd.sandwich_norm_fwd(s["x"], s["residual"], s["residual_out"], s["post"], gate=s["gate"], residual_scale=c["scale"],
                             gain=s["gain"] if c["out"] != "none" else None, out=s["out"], out_scale=s["out_scale"], eps=_EPS)
        out = {"residual_out": s["residual_out"]}
        if c["out"] != "none":
            out["out"] = s["out"]
        return {**out, "scale": s["out_scale"]} if c["out"] == "fp8" else out
    if c["op"] == "linear":
        bd.linear_w4_fwd(s["x"], s["w"], s["bias"], s["y"], group=c["group"], act=c["act"], gate=s["gate"], residual=s["residual"])
        return s["y"]
    if c["op"] == "append":
        bd.cache4_append(s["k"], s["v"], s["cache"], kv_len=s["kv_len"])
        bd.cache4_read(s["cache"], s["k_back"], s["v_back"], kv_len=s["kv_len"])
        return [s["k_back"], s["v_back"]]
    bd.sdpa_cache4_fwd(s["q"], s["cache"], s["out"], c["heads"], window=c["window"], sinks=c["sinks"], kv_len=s["kv_len"],
                       key_mask=s["key_mask"])
    return s["out"]


def _visible(case):
    """(query, key) pairs, and cache rows that some query sees, over the batch."""
    new, window, sinks, padded = case["new"], case["window"], case["sinks"], case["padded"]
    pairs = rows = 0
    for n in _lengths(case):
        for p in range(max(0, n - new), n):
            first = max(0, p - window + 1) if window else 0
            pairs += max(0, p + 1 - max(first, padded)) + max(0, min(sinks, first) - padded)
        first = max(0, n - new - window + 1) if window else 0
        rows += max(0, n - max(first, padded)) + max(0, min(sinks, first) - padded)
    return pairs, rows


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        out = {"none": 0, "same": 2 * n, "fp8": n + 4 * case["rows"]}[case["out"]]
        vectors = 1 + case["gates"] + (case["out"] != "none")
        return {"bytes": 6 * n + 2 * case["cols"] * vectors + out, "flops": 12 * n}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": n * k // 2 + 4 * n * -(-k // case["group"]) + 2 * m * k + 2 * n * (case["bias"] + case["gate"]) +
                2 * m * n * (1 + case["residual"]), "flops": 2 * m * n * k}
    nkv, hd = case["kv_heads"], case["head_dim"]
    held = 2 * nkv * (hd // 2 + 4 * hd // case["group"])       # bytes of a row of K and V
    if case["op"] == "append":
        n = case["batch"] * case["new"]
        return {"bytes": n * (8 * nkv * hd + held) + 4 * case["batch"] * case["ragged"], "flops": 12 * n * nkv * hd}
    pairs, rows = _visible(case)
    q = case["batch"] * case["new"] * case["heads"] * hd
    extra = 4 * case["batch"] * case["ragged"] + (4 * case["rows"] if case["padded"] else 0)
    return {"bytes": 4 * q + rows * held + extra, "flops": 4 * pairs * case["heads"] * hd}


# ------------------------------------------- the definitions, in 64 bits
def _exact_held(x, group):
    """The values that 4-bit groups of x stand for, from the definition."""
    g = x.double().unflatten(-1, (-1, group))
    low = g.min(-1, keepdim=True).values
    step = (g.max(-1, keepdim=True).values.sub(low) / 15).to(x.dtype).double()
    code = torch.nan_to_num((g - low) / step).round().clamp(0, 15)
    return (low + step * code).flatten(-2)


def _exact_cache(case, s):
    new, hd, share = case["new"], case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    for b, n in enumerate(_lengths(case)):
        i = torch.arange(n - new, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        hidden = (j > i) | (j < case["padded"])
        if case["window"]:
            hidden |= (i - j >= case["window"]) & (j >= case["sinks"])
        empty = hidden.all(1)
        for kv in range(case["kv_heads"]):
            at = slice(kv * hd, (kv + 1) * hd)
            k, v = (_exact_held(s[x][b, :n, at], case["group"]) for x in ("k", "v"))
            for h in range(kv * share, (kv + 1) * share):
                cols = slice(h * hd, (h + 1) * hd)
                a = s["q"][b, :, cols].double() @ k.T / math.sqrt(hd)
                a = torch.softmax(a.masked_fill_(hidden, -math.inf), 1).masked_fill_(empty[:, None], 0)
                out[b, :, cols] = a @ v
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        branch = s["post"].double() * x / (x.square().sum(1, keepdim=True) / case["cols"] + _EPS).sqrt()
        if s["gate"] is not None:
            branch *= s["gate"].double().repeat_interleave(case["rows"] // case["gates"], 0)
        h = branch + case["scale"] * s["residual"].double()
        if case["out"] == "none":
            return {"residual_out": h}
        y = s["gain"].double() * h / (h.square().sum(1, keepdim=True) / case["cols"] + _EPS).sqrt()
        if case["out"] == "same":
            return {"residual_out": h, "out": y}
        scale = y.abs().max(1).values / _E4M3_MAX
        return {"residual_out": h, "out": y / scale[:, None], "scale": scale}
    if case["op"] == "linear":
        low, high = s["codes"] % 16, s["codes"] // 16
        codes = torch.empty(case["outputs"], case["inputs"], device="cuda", dtype=torch.float64)
        codes[:, ::2], codes[:, 1::2] = low, high
        step, least = (s["scales"][..., i].double().repeat_interleave(case["group"], 1)[:, :case["inputs"]] for i in (0, 1))
        z = torch.mm(s["x"].double(), (codes * step + least).T)
        if s["bias"] is not None:
            z = z + s["bias"].double()
        if case["act"] == "gelu":
            z = z * torch.special.ndtr(z)
        elif case["act"] == "gelu_tanh":
            z = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
        elif case["act"] == "silu":
            z = z * torch.sigmoid(z)
        if s["gate"] is not None:
            z = s["gate"].double() * z
        return z if s["residual"] is None else s["residual"].double() + z
    if case["op"] == "append":
        return [_exact_held(s[x], case["group"]) for x in ("k", "v")]
    return _exact_cache(case, s)
