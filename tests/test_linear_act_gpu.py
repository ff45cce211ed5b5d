"""Projection with scales, bias, activation, gate and residual in the epilogue, against the formula in 64 bits.

Tolerance of y = r + g act(z): the output's rounding u |y|, with u = 2^-8 (BF16) or 2^-11 (FP16); z is a sum of K
products in K / 16 steps, each off by at most 2^-23 of the partial sum, which for the inputs here stays below a
quarter of S = sum |x w|: for K up to 10240 below 2^-15 S; the activations' slopes are at most 1.13 and their own
error below 4e-6 |z|."""
import pytest
import torch

from layer_shapes import SHAPES

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn
ACT = {"none": lambda z: z, "gelu": lambda z: z * torch.special.ndtr(z), "silu": lambda z: z * torch.sigmoid(z),
       "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))}


def randn(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    return (scale * torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))).to(dtype)


def e4m3(t):
    s = t.float().abs().amax(1).clamp_min(1e-6) / 448
    return (t.float() / s[:, None]).to(E4M3), s


def problem(seed, M, N, K, dtype=torch.bfloat16, fp8=False, bias=True, gate=False, residual=False):
    x, w = randn(seed, M, K, dtype=dtype), randn(seed + 1, N, K, dtype=dtype, scale=2 / K ** 0.5)
    p = {"x": x, "w": w, "bias": None, "gate": None, "residual": None, "x_scale": None, "w_scale": None, "dtype": dtype}
    if fp8:
        p["x"], p["x_scale"] = e4m3(x)
        p["w"], p["w_scale"] = e4m3(w)
    if bias:
        p["bias"] = randn(seed + 2, N, dtype=dtype)
    if gate:
        p["gate"] = randn(seed + 3, N, dtype=dtype)
    if residual:
        p["residual"] = randn(seed + 4, M, N, dtype=dtype)
    return p


def formula(p, act):
    x, w = p["x"].double(), p["w"].double()
    z, S = x @ w.T, x.abs() @ w.abs().T
    if p["x_scale"] is not None:
        z, S = z * p["x_scale"].double()[:, None], S * p["x_scale"].double()[:, None]
    if p["w_scale"] is not None:
        z, S = z * p["w_scale"].double(), S * p["w_scale"].double()
    if p["bias"] is not None:
        z = z + p["bias"].double()
    y, err = ACT[act](z), 1.13 * 2.0 ** -15 * S + 4e-6 * z.abs()
    if p["gate"] is not None:
        y, err = y * p["gate"].double(), err * p["gate"].double().abs()
    if p["residual"] is not None:
        y = y + p["residual"].double()
    return y, UNIT[p["dtype"]] * y.abs() + (1 + UNIT[p["dtype"]]) * err + 1e-7


def call(bd, p, act, y=None, **kw):
    if y is None:
        y = torch.full((p["x"].shape[0], p["w"].shape[0]), float("nan"), device="cuda", dtype=p["dtype"])
    bd.linear_act_fwd(p["x"], p["w"], p["bias"], y, act=act, gate=p["gate"], residual=p["residual"], x_scale=p["x_scale"],
                      w_scale=p["w_scale"], **kw)
    assert bd.device_status() == 0
    return y


def check(y, p, act):
    ref, bound = formula(p, act)
    err = (y.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, first {bad.nonzero()[0].tolist()}, " \
        f"worst {float((err / bound).nan_to_num(1e9).max()):.3g} times the bound"


SIZES = [(1, 8, 16), (1, 2560, 1280), (3, 24, 48), (8, 5120, 5120), (16, 72, 2560), (17, 1288, 640), (64, 1280, 1280), (65, 1288, 656),
         (127, 200, 96), (128, 128, 128), (129, 136, 144), (256, 1280, 5120), (333, 1288, 656), (511, 5120, 320), (600, 640, 2560),
         (1024, 2560, 640), (1500, 2304, 2240), (2166, 2560, 1040), (4096, 320, 320), (300, 8, 10240), (5, 10240, 16)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
def test_sizes(bd, M, N, K, kind):
    dtype = torch.float16 if kind == "fp16" else torch.bfloat16
    p = problem(M + N + K, M, N, K, dtype, kind == "fp8", residual=True)
    check(call(bd, p, "none"), p, "none")
    p = problem(M + N + K + 9, M, N, K, dtype, kind == "fp8", gate=True, residual=True)
    check(call(bd, p, "gelu_tanh"), p, "gelu_tanh")


@pytest.mark.parametrize("M,N,K,act,kernel,cols,split", SHAPES)
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
def test_every_tile_width_and_split(bd, M, N, K, act, kernel, cols, split, kind):
    p = problem(M + N + K, M, N, 2 * K if kind == "fp8" else K, torch.float16 if kind == "fp16" else torch.bfloat16, kind == "fp8", True, True, True)
    name = "gelu" if act else "none"
    check(call(bd, p, name), p, name)


# up to 16 rows: one and two eights of them; many rows of W with a short K and a long one, few with K over two, four and eight
# CTAs; K with a remainder of a turn of 64
@pytest.mark.parametrize("N,K", [(7200, 64), (7200, 640), (8192, 2560), (64, 10240), (1280, 5120), (640, 2560), (72, 4112), (2560, 2576), (24, 16), (8, 8208)])
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
def test_few_rows(bd, M, N, K, kind):
    p = problem(M + N + K, M, N, K, torch.float16 if kind == "fp16" else torch.bfloat16, kind == "fp8", True, M % 2 == 0, True)
    check(call(bd, p, "silu"), p, "silu")


# one row tile with fewer rows than the MMA reads: several tiles to an SM (a short ring, a ring of two), one (the longest
# ring, more turns than it has slots), K over two and eight CTAs
@pytest.mark.parametrize("N,K", [(9600, 208), (9600, 640), (2080, 2064), (2528, 1280), (72, 2560)])
@pytest.mark.parametrize("M", [17, 25, 56, 65, 120, 127])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
def test_one_row_tile(bd, M, N, K, kind):
    p = problem(M + N + K, M, N, K, torch.float16 if kind == "fp16" else torch.bfloat16, kind == "fp8", True, True, True)
    check(call(bd, p, "gelu"), p, "gelu")


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("bias,gate,residual", [(b, g, r) for b in (0, 1) for g in (0, 1) for r in (0, 1)])
@pytest.mark.parametrize("M,N,K", [(2, 512, 320), (40, 264, 1280), (700, 768, 256), (1300, 2560, 512)])
def test_every_combination(bd, M, N, K, act, bias, gate, residual):
    for kind in ("bf16", "fp8"):
        p = problem(M, M, N, K, torch.bfloat16, kind == "fp8", bias, gate, residual)
        check(call(bd, p, act), p, act)
    p = problem(M, M, N, K, torch.float16, True, bias, gate, residual)        # 8-bit operands, FP16 output
    check(call(bd, p, act), p, act)


@pytest.mark.parametrize("M", [1, 30, 900])
def test_scales_are_optional(bd, M):
    p = problem(1, M, 512, 256, fp8=True, residual=True)
    for drop in (("x_scale",), ("w_scale",), ("x_scale", "w_scale")):
        q = dict(p, **{k: None for k in drop})
        check(call(bd, q, "none"), q, "none")


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_over_their_range(bd, act):
    """z from -60 to 60 and far beyond, one value to a column through the bias."""
    n = 4096
    p = problem(2, 3, n, 64, torch.float16, residual=False)
    p["x"].zero_()
    p["bias"] = torch.cat([torch.linspace(-60, 60, n - 8), torch.tensor([-6e4, -1e3, -100.0, 0.0, 1e-4, 100.0, 1e3, 6e4])]).cuda().half()
    check(call(bd, p, act), p, act)
    q = dict(p, dtype=torch.bfloat16, x=p["x"].bfloat16(), w=p["w"].bfloat16(), bias=(p["bias"].bfloat16() * 1e30))
    y = call(bd, q, act)
    assert torch.isfinite(y).all() and (y[:, q["bias"] > 0] == q["bias"][q["bias"] > 0]).all() and (y[:, q["bias"] < 0].abs() < 1e-3).all()


@pytest.mark.parametrize("M,N,K", [(4, 264, 640), (33, 128, 1280), (150, 200, 64), (2100, 512, 640)])
@pytest.mark.parametrize("fp8", [False, True])
def test_strides_and_the_residual_in_place(bd, M, N, K, fp8):
    p = problem(5, M, N, K, fp8=fp8, residual=True)
    want = call(bd, p, "silu")
    wide = {"x": (M, K + 32), "w": (N, K + 16), "residual": (M, N + 24)}
    q = dict(p)
    for name, shape in wide.items():
        t = torch.zeros(shape, device="cuda").to(p[name].dtype)
        at = 16 if name != "residual" else 8
        at = 0 if name == "w" else at
        t[:, at:at + p[name].shape[1]] = p[name]
        q[name] = t[:, at:at + p[name].shape[1]]
    y = torch.full((M + 2, N + 40), 7.0, device="cuda", dtype=torch.bfloat16)
    call(bd, q, "silu", y[1:-1, 16:16 + N])
    assert (y[1:-1, 16:16 + N] == want).all()
    y[1:-1, 16:16 + N] = 7
    assert (y == 7).all()
    r = p["residual"].clone()
    call(bd, dict(p, residual=r), "silu", r)
    assert (r == want).all()


def test_rows_that_are_not_finite_stay_where_they_are(bd):
    for M, N in ((20, 512), (600, 768)):
        p = problem(6, M, N, 640, residual=True)
        good = call(bd, p, "none")
        p["x"][3, 100] = float("nan")
        p["x"][7, 11] = float("inf")
        p["residual"][9, 5] = float("inf")
        y = call(bd, p, "none")
        assert torch.isnan(y[3]).all() and not torch.isfinite(y[7]).any() and torch.isinf(y[9, 5])
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[[3, 7]] = False
        keep[9, 5] = False
        assert (y[keep] == good[keep]).all()


def test_offsets_past_32_bits(bd):
    """An output and a residual whose last rows lie beyond 2^31 elements."""
    M, N, K, ld = 36000, 64, 32, 65536
    p = problem(7, M, N, K, residual=False)
    y = torch.zeros(M, ld, device="cuda", dtype=torch.bfloat16)
    p["residual"] = y[:, 512:512 + N]
    p["residual"].copy_(randn(1, M, N))
    q = dict(p, residual=p["residual"].clone())
    call(bd, p, "none", y[:, :N])
    check(y[:, :N], q, "none")


def test_no_rows_streams_and_repeats(bd):
    p = problem(8, 5, 640, 320, residual=True)
    bd.linear_act_fwd(p["x"][:0], p["w"], p["bias"], torch.empty(0, 640, device="cuda", dtype=torch.bfloat16))
    for M, N, K in ((5, 640, 1280), (1000, 1280, 640)):
        p = problem(8, M, N, K, residual=True)
        a = call(bd, p, "gelu")
        side, b = torch.cuda.Stream(), torch.empty_like(a)
        torch.cuda.synchronize()
        call(bd, p, "gelu", b, stream=side)
        side.synchronize()
        assert (a == b).all()


def test_behind_the_norm(bd):
    """Rows in 8 bits straight from the norm, both calls on one stream."""
    M, N, K = 300, 1280, 640
    h, g = randn(1, M, K), 1 + randn(2, K, scale=0.02)
    p = problem(9, M, N, K, fp8=True)
    p["x"], p["x_scale"] = torch.empty(M, K, device="cuda", dtype=E4M3), torch.empty(M, device="cuda")
    bd.add_rmsnorm_fwd(h, p["x"], g, out_scale=p["x_scale"])
    check(call(bd, p, "silu"), p, "silu")


def test_graph_capture(bd):
    for M in (3, 800):
        p = problem(10, M, 768, 640, residual=True, gate=True)
        y = call(bd, p, "gelu")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            bd.linear_act_fwd(p["x"], p["w"], p["bias"], y, act="gelu", gate=p["gate"], residual=p["residual"])
        p["x"].copy_(randn(11, M, 640))
        g.replay()
        torch.cuda.synchronize()
        check(y, p, "gelu")


def test_refusals(bd):
    p = problem(12, 4, 64, 64, residual=True, gate=True)
    y = torch.full((4, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    f32 = torch.ones(64, device="cuda")
    x8, xs = e4m3(p["x"])
    w8, ws = e4m3(p["w"])

    def refuse(x=p["x"], w=p["w"], bias=p["bias"], out=y, **kw):
        with pytest.raises(bd.BdattnError):
            bd.linear_act_fwd(x, w, bias, out, **kw)
    refuse(act="relu6")
    refuse(act=1)
    refuse(x=p["x"].half())
    refuse(w=p["w"].half())
    refuse(x=p["x"].half(), w=p["w"].half())
    refuse(x=x8)
    refuse(x=p["x"][:, :32])
    refuse(x=p["x"][:, :60], w=p["w"][:, :60])
    refuse(x=x8[:, :56], w=w8[:, :56])                              # 8-bit rows: multiples of 16
    refuse(x=p["x"].t())
    refuse(bias=p["bias"][:32])
    refuse(bias=p["bias"].float())
    refuse(gate=p["gate"].half())
    refuse(residual=p["residual"][:2])
    refuse(residual=p["residual"].half())
    refuse(out=y[:2])
    refuse(out=y.float())
    refuse(out=torch.empty(4, 72, device="cuda", dtype=torch.bfloat16)[:, 4:68])          # 8-byte aligned
    refuse(x_scale=xs)                                              # scales of 16-bit rows
    refuse(x=x8, w=w8, x_scale=xs[:3], w_scale=ws)
    refuse(x=x8, w=w8, x_scale=xs.half(), w_scale=ws)
    refuse(x=x8, w=w8, x_scale=xs, w_scale=f32[:4])
    refuse(w=p["w"][:60], bias=p["bias"][:60], out=y[:, :60])       # width: a multiple of 8
    c = bd.LinearActParams(dtype=bd.BF16, in_dtype=bd.BF16, M=4, N=64, K=64, x=p["x"].data_ptr(), w=p["w"].data_ptr(), y=y.data_ptr(), act=9)
    L = bd.lib()
    assert L.bdattn_linear_act_fwd(c, None) == -1 and "activation" in bd.last_error()
    c.act, c.y_ld = 0, 32
    assert L.bdattn_linear_act_fwd(c, None) == -1 and "stride" in bd.last_error()
    c.y_ld, c.residual, c.residual_ld = 0, p["residual"].data_ptr(), 60
    assert L.bdattn_linear_act_fwd(c, None) == -1 and "residual" in bd.last_error()
    c.residual, c.x = None, None
    assert L.bdattn_linear_act_fwd(c, None) == -1 and "null" in bd.last_error()
    assert L.bdattn_linear_act_fwd(None, None) == -1
    assert (y == 7).all()
