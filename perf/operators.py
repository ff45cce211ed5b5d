"""The operators of a causal pre-norm layer over a stream of tokens, as timed cases.

    norm     residual addition + RMSNorm of rows, to 16 bits or to 8 bits (e4m3)
             with a scale per row: what stands in front of every projection
    linear   X W^T with scales of 8-bit operands, bias, activation, gate and residual
             in the epilogue: the projections and the feed-forward layers
    window   causal attention over a cache with a sliding window and a few first
             tokens that stay visible: prefill, a chunk of new rows, single tokens

Activations are N(0, 1), weights N(0, 0.02), gains 1 + N(0, 0.02), as everywhere in
this repository's tests and benchmark.
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
        # One new token: a single row, 8-bit output for the projection behind it: latency.
        {"name": "norm_one_token", "op": "norm", "rows": 1, "cols": 2560, "residual": True, "out": "fp8", "dtype": "bf16"},
        # Rows of an odd width without a residual (the first norm of a stream), 16-bit output.
        {"name": "norm_odd_columns", "op": "norm", "rows": 777, "cols": 1365, "residual": False, "out": "same",
         "dtype": "fp16"},
        # A long prompt at 5120 columns, residual updated, 8-bit output: bound by memory.
        {"name": "norm_long", "op": "norm", "rows": 16384, "cols": 5120, "residual": True, "out": "fp8", "dtype": "bf16"},
        # Eight sequences' single tokens against 8-bit weights: the weights' bytes are the time.
        {"name": "linear_tokens_fp8", "op": "linear", "rows": 8, "inputs": 5120, "outputs": 5120, "act": "none",
         "bias": True, "gate": False, "residual": True, "type": "fp8"},
        # One token through a 16-bit projection with activation.
        {"name": "linear_one_token", "op": "linear", "rows": 1, "inputs": 2560, "outputs": 5120, "act": "silu",
         "bias": True, "gate": False, "residual": False, "type": "bf16"},
        # A short ragged prompt, sizes that no tile divides.
        {"name": "linear_ragged", "op": "linear", "rows": 333, "inputs": 648, "outputs": 1288, "act": "gelu",
         "bias": True, "gate": False, "residual": True, "type": "fp16"},
        # Down projection of a feed-forward layer, gated into the residual stream (rows of a portrait image).
        {"name": "linear_down_gated", "op": "linear", "rows": 2166, "inputs": 10240, "outputs": 2560, "act": "none",
         "bias": True, "gate": True, "residual": True, "type": "bf16"},
        # Up projection with the tanh GELU from 8-bit rows and weights: the most arithmetic of a layer.
        {"name": "linear_up_fp8", "op": "linear", "rows": 4096, "inputs": 2560, "outputs": 10240, "act": "gelu_tanh",
         "bias": True, "gate": False, "residual": False, "type": "fp8"},
        # One sequence, one token, a short cache: latency.
        {"name": "window_one_token", "op": "window", "batch": 1, "new": 1, "cache": 777, "heads": 24, "kv_heads": 8,
         "head_dim": 128, "window": 512, "sinks": 4, "ragged": False, "padded": 0, "dtype": "bf16"},
        # A serving batch of single tokens over caches of different lengths: the visible rows' bytes are the time.
        {"name": "window_tokens_ragged", "op": "window", "batch": 32, "new": 1, "cache": 32768, "heads": 24,
         "kv_heads": 8, "head_dim": 128, "window": 4096, "sinks": 64, "ragged": True, "padded": 0, "dtype": "bf16"},
        # Prefill of a left-padded prompt (its first rows see nothing), heads of 64.
        {"name": "window_prefill_padded", "op": "window", "batch": 2, "new": 2166, "cache": 2166, "heads": 8,
         "kv_heads": 8, "head_dim": 64, "window": 300, "sinks": 150, "ragged": False, "padded": 141, "dtype": "fp16"},
        # Prefill of a long stream, grouped heads.
        {"name": "window_prefill_long", "op": "window", "batch": 1, "new": 8192, "cache": 8192, "heads": 24,
         "kv_heads": 8, "head_dim": 128, "window": 2048, "sinks": 64, "ragged": False, "padded": 0, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "window"])
    if op == "norm":
        cols = _log_int(rng, 64, 8192)
        if rng.random() < 0.75:
            cols = (cols + 7) // 8 * 8
        return {"op": op, "rows": _log_int(rng, 1, max(2, min(16384, 16384 * 5120 // cols))), "cols": cols,
                "residual": rng.random() < 0.7, "out": rng.choice(["same", "fp8"]), "dtype": rng.choice(["bf16", "fp16"])}
    if op == "linear":
        kind = rng.choice(["bf16", "fp16", "fp8"])
        step = 16 if kind == "fp8" else 8
        inputs, outputs = (step * _log_int(rng, 64 // step, 10240 // step) for _ in range(2))
        rows = _log_int(rng, 1, min(4096, 4096 * 10240 * 2560 // (inputs * outputs)))
        return {"op": op, "rows": rows, "inputs": inputs, "outputs": outputs,
                "act": rng.choice(["none", "none", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.7,
                "gate": rng.random() < 0.3, "residual": rng.random() < 0.5, "type": kind}
    group, kv_heads = rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([40, 64, 80, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    window, sinks = rng.choice([0, _log_int(rng, 16, 4096)]), rng.choice([0, 4, _log_int(rng, 1, 256)])
    if rng.random() < 0.5:                                 # a few new tokens of several sequences
        batch = _log_int(rng, 1, 32)
        return {"op": op, "batch": batch, "new": rng.choice([1, 1, 1, rng.randint(2, 8)]),
                "cache": _log_int(rng, 16, 32768 // batch if window == 0 else 32768), "heads": group * kv_heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "window": window, "sinks": sinks,
                "ragged": rng.random() < 0.7, "padded": 0, "dtype": dtype}
    most = int(8192 * math.sqrt(24 / (group * kv_heads)))  # rows whose score matrix is no larger than the longest case's
    cache = _log_int(rng, 65, min(most, 16384) if window else min(most, 8192) // 2)
    batch = 2 if cache < 3000 and rng.random() < 0.4 else 1
    new = cache if rng.random() < 0.6 else rng.randint(min(64, cache), cache)
    return {"op": op, "batch": batch, "new": new, "cache": cache, "heads": group * kv_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "window": window, "sinks": sinks, "ragged": rng.random() < 0.3,
            "padded": rng.choice([0, 0, rng.randint(1, 40)]), "dtype": dtype}


class _Make:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def act(self, dtype, *shape):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=self.gen)


def _e4m3(t):
    """Rows in 8 bits and their FP32 scales."""
    scale = t.float().abs().amax(1) / _E4M3_MAX
    return (t.float() / scale[:, None]).to(torch.float8_e4m3fn), scale


def _lengths(case):
    """Filled rows of each sequence's cache."""
    cache, new = case["cache"], case["new"]
    if not case["ragged"]:
        return [cache] * case["batch"]
    return [max(new, cache - (b * 2654435761 % 4096) * (cache - cache // 3) // 4096) for b in range(case["batch"])]


def prepare(case, seed):
    m = _Make(seed)
    if case["op"] == "norm":
        dtype, shape = _DTYPES[case["dtype"]], (case["rows"], case["cols"])
        s = {"case": case, "x": m.act(dtype, *shape), "gain": 1 + 0.02 * m.act(dtype, case["cols"]), "residual": None,
             "residual_out": None, "out": torch.empty(shape, device="cuda", dtype=dtype), "scale": None}
        if case["residual"]:
            s["residual"] = m.act(dtype, *shape)
            s["residual_out"] = torch.empty_like(s["x"])
        if case["out"] == "fp8":
            s["out"] = torch.empty(shape, device="cuda", dtype=torch.float8_e4m3fn)
            s["scale"] = torch.empty(case["rows"], device="cuda")
        return s
    if case["op"] == "linear":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        fp8 = case["type"] == "fp8"
        dtype = torch.bfloat16 if fp8 else _DTYPES[case["type"]]
        x, w = m.act(dtype, rows, inputs), 0.02 * m.act(dtype, outputs, inputs)
        s = {"case": case, "x_scale": None, "w_scale": None, "bias": None, "gate": None, "residual": None,
             "y": torch.empty(rows, outputs, device="cuda", dtype=dtype)}
        if fp8:
            x, s["x_scale"] = _e4m3(x)
            w, s["w_scale"] = _e4m3(w)
        s["x"], s["w"] = x, w
        if case["bias"]:
            s["bias"] = 0.02 * m.act(dtype, outputs)
        if case["gate"]:
            s["gate"] = 0.5 * m.act(dtype, outputs)
        if case["residual"]:
            s["residual"] = m.act(dtype, rows, outputs)
        return s
    dtype, b, hd = _DTYPES[case["dtype"]], case["batch"], case["head_dim"]
    s = {"case": case, "q": m.act(dtype, b, case["new"], case["heads"] * hd),
         "k": m.act(dtype, b, case["cache"], case["kv_heads"] * hd),
         "v": m.act(dtype, b, case["cache"], case["kv_heads"] * hd), "kv_len": None, "key_mask": None}
    s["out"] = torch.empty_like(s["q"])
    if case["ragged"]:
        s["kv_len"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    if case["padded"]:
        s["key_mask"] = (torch.arange(case["cache"], device="cuda") >= case["padded"]).float()
    return s


# ------------------------------------------------------------- plain forms
def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS) * s["gain"].float()
    out = {} if s["residual"] is None else {"residual_out": h.to(s["x"].dtype)}
    if s["scale"] is None:
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
    z = s["x"].float() @ s["w"].float().t()
    if s["x_scale"] is not None:
        z = z * s["x_scale"][:, None] * s["w_scale"]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _plain_act(z, s["case"]["act"])
    if s["gate"] is not None:
        y = y * s["gate"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["y"].dtype)


def _plain_window(s):
    c = s["case"]
    b, new, cache, nkv, hd = c["batch"], c["new"], c["cache"], c["kv_heads"], c["head_dim"]
    q = s["q"].float().view(b, new, nkv, c["heads"] // nkv, hd)
    k, v = s["k"].float().view(b, cache, nkv, hd), s["v"].float().view(b, cache, nkv, hd)
    key = torch.arange(cache, device="cuda")
    length = s["kv_len"].long() if s["kv_len"] is not None else torch.full((b,), cache, device="cuda")
    pos = (length - new)[:, None] + torch.arange(new, device="cuda")
    seen = key <= pos[:, :, None]
    if c["window"]:
        seen = seen & ((key > pos[:, :, None] - c["window"]) | (key < c["sinks"]))
    if s["key_mask"] is not None:
        seen = seen & (s["key_mask"] != 0)
    score = torch.einsum("bihgd,bjhd->bhgij", q, k) * (1 / math.sqrt(hd))
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0))
    total = p.sum(-1)
    p = p / torch.where(total > 0, total, 1)[..., None]
    return torch.einsum("bhgij,bjhd->bihgd", p, v).reshape(s["q"].shape).to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "window": _plain_window}[c["op"]](s)
    import brodiffusion_b200 as bd
    if c["op"] == "norm":
        bd.add_rmsnorm_fwd(s["x"], s["out"], s["gain"], residual=s["residual"], residual_out=s["residual_out"],
                           out_scale=s["scale"], eps=_EPS)
        out = {} if s["residual"] is None else {"residual_out": s["residual_out"]}
        return {**out, "out": s["out"]} if s["scale"] is None else {**out, "out": s["out"], "scale": s["scale"]}
    if c["op"] == "linear":
        bd.linear_act_fwd(s["x"], s["w"], s["bias"], s["y"], act=c["act"], gate=s["gate"], residual=s["residual"],
                          x_scale=s["x_scale"], w_scale=s["w_scale"])
        return s["y"]
    bd.sdpa_window_fwd(s["q"], s["k"], s["v"], s["out"], c["heads"], window=c["window"], sinks=c["sinks"],
                       num_kv_heads=c["kv_heads"], kv_len=s["kv_len"], key_mask=s["key_mask"])
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
        out = n + 4 * case["rows"] if case["out"] == "fp8" else 2 * n
        return {"bytes": 2 * n + (4 * n if case["residual"] else 0) + 2 * case["cols"] + out, "flops": 6 * n}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        size = 1 if case["type"] == "fp8" else 2
        extra = 4 * (m + n) if case["type"] == "fp8" else 0
        return {"bytes": size * k * (m + n) + extra + 2 * n * (case["bias"] + case["gate"]) +
                2 * m * n * (1 + case["residual"]), "flops": 2 * m * n * k}
    pairs, rows = _visible(case)
    hd, q = case["head_dim"], case["batch"] * case["new"] * case["heads"] * case["head_dim"]
    extra = 4 * case["batch"] * case["ragged"] + (4 * case["cache"] if case["padded"] else 0)
    return {"bytes": 4 * q + 4 * rows * case["kv_heads"] * hd + extra, "flops": 4 * pairs * case["heads"] * hd}


# ------------------------------------------- the definitions, in 64 bits
def _exact_window(s):
    c = s["case"]
    new, hd, group = c["new"], c["head_dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    for b, n in enumerate(_lengths(c)):
        i = torch.arange(n - new, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        hidden = (j > i) | (j < c["padded"])
        if c["window"]:
            hidden |= (i - j >= c["window"]) & (j >= c["sinks"])
        empty = hidden.all(1)
        for h in range(c["heads"]):
            cols, kv = slice(h * hd, (h + 1) * hd), slice(h // group * hd, (h // group + 1) * hd)
            a = s["q"][b, :, cols].double() @ s["k"][b, :n, kv].double().T / math.sqrt(hd)
            a = torch.softmax(a.masked_fill_(hidden, -math.inf), 1).masked_fill_(empty[:, None], 0)
            out[b, :, cols] = a @ s["v"][b, :n, kv].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        y = s["gain"].double() * h / (h.square().sum(1, keepdim=True) / case["cols"] + _EPS).sqrt()
        out = {} if s["residual"] is None else {"residual_out": h}
        if s["scale"] is None:
            return {**out, "out": y}
        scale = y.abs().max(1).values / _E4M3_MAX
        return {**out, "out": y / scale[:, None], "scale": scale}
    if case["op"] == "linear":
        z = torch.mm(s["x"].double(), s["w"].double().T)
        if s["x_scale"] is not None:
            z = z * torch.outer(s["x_scale"].double(), s["w_scale"].double())
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
    return _exact_window(s)
