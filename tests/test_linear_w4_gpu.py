"""Products with 4-bit weights against their formula in 64 bits.

Tolerance.  The weights are exact, so what is lost is the FP32 part and one rounding.  Products of X and a code are exact; a
sum of 32 of them, the sum of X beside it and their scaling take a few steps of 2^-23 (mma.sync cuts off) of
sum |x| (15 step + |low|), and a warp adds up at most K / 256 of those, the warps and CTAs at most 64 more:
(K / 128 + 32) 2^-23 of that sum in all.  An activation's slope is at most 1.13, its own error below 1e-6."""
import pytest
import torch

from four_bit import UNIT, packed_pairs, quantised, randn, values

pytestmark = pytest.mark.gpu

TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}       # half of the smallest step


def weights(seed, n, k, group, dtype):
    """Codes and pairs of a random matrix; columns beyond K are there for the last group alone."""
    whole = -(-k // group) * group
    codes, scales = quantised(randn(seed, n, whole, dtype=dtype, scale=0.02), group)
    return codes[:, :k], scales


def pack(bd, codes, scales, group):
    n, k = codes.shape
    guard = torch.full((bd.w4_bytes(n, k, group) + 64,), 0xa5, device="cuda", dtype=torch.uint8)
    bd.w4_pack(packed_pairs(codes), scales, guard[:-64], group=group)
    assert (guard[-64:] == 0xa5).all()
    return guard[:-64]


def activation(z, act):
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid((8 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if act == "silu" else z


def check(y, x, codes, scales, group, bias=None, gate=None, residual=None, act="none"):
    w, xd = values(codes, scales, group), x.double()
    s = scales.double().repeat_interleave(group, 1)[:, :codes.shape[1]]
    size = xd.abs() @ (15 * s[..., 0].abs() + s[..., 1].abs()).T
    z = xd @ w.T
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    a = activation(z, act)
    g = gate.double() if gate is not None else torch.ones_like(a[0])
    r = residual.double() if residual is not None else torch.zeros_like(a)
    ref = r + g * a
    fp32 = (x.shape[1] / 128 + 32) * 2.0 ** -23 * 1.13 * size * g.abs() + 1e-6 * ((g * a).abs() + r.abs())
    err = (y.double() - ref).abs()
    bad = ~(err <= UNIT[x.dtype] * ref.abs() + fp32 + TINY[x.dtype])
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / (UNIT[x.dtype] * ref.abs() + fp32)).max()):.3g} of the tolerance"


def run(bd, x, packed, n, group, bias=None, **kw):
    y = torch.full((x.shape[0], n), float("nan"), device="cuda", dtype=x.dtype)
    bd.linear_w4_fwd(x, packed, bias, y, group=group, **kw)
    assert bd.device_status() == 0
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 8), (16, 128), (17, 136), (100, 648), (1291, 1368), (320, 2560), (33, 10240), (5000, 264)])
def test_sizes(bd, n, k, group, dtype):
    codes, scales = weights(n + k, n, k, group, dtype)
    packed = pack(bd, codes, scales, group)
    for m in (1, 2, 7, 8, 9, 16, 17, 33, 64):
        x = randn(m, m, k, dtype=dtype)
        check(run(bd, x, packed, n, group), x, codes, scales, group)


@pytest.mark.parametrize("m", [65, 130, 1000])
def test_more_rows_than_a_pass_takes(bd, m):
    codes, scales = weights(1, 200, 520, 32, torch.bfloat16)
    x = randn(m, m, 520)
    check(run(bd, x, pack(bd, codes, scales, 32), 200, 32), x, codes, scales, 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("parts", range(8))
def test_what_stands_behind_the_product(bd, parts, act, dtype):
    n, k, group = 130, 392, 64
    codes, scales = weights(7, n, k, group, dtype)
    packed = pack(bd, codes, scales, group)
    for m in (1, 12, 40):
        x = randn(m, m, k, dtype=dtype, scale=3.0)
        bias = randn(2, n, dtype=dtype) if parts & 1 else None
        gate = randn(3, n, dtype=dtype) if parts & 2 else None
        residual = randn(4, m, n, dtype=dtype) if parts & 4 else None
        y = run(bd, x, packed, n, group, bias, act=act, gate=gate, residual=residual)
        check(y, x, codes, scales, group, bias, gate, residual, act)


@pytest.mark.parametrize("m", [3, 11, 50])
def test_rows_inside_wider_tensors_and_the_residual_in_place(bd, m):
    n, k, group = 77, 264, 32
    codes, scales = weights(5, n, k, group, torch.bfloat16)
    packed = pack(bd, codes, scales, group)
    x, wide = randn(1, m, k + 24)[:, 8:8 + k], randn(2, m, n + 9)
    before, y = wide.clone(), wide[:, 5:5 + n]
    bd.linear_w4_fwd(x, packed, None, y, group=group, residual=y)
    check(y, x, codes, scales, group, residual=before[:, 5:5 + n])
    assert (wide[:, :5] == before[:, :5]).all() and (wide[:, 5 + n:] == before[:, 5 + n:]).all()


def test_codes_and_pairs_inside_wider_tensors(bd):
    n, k, group = 40, 264, 32
    codes, scales = weights(6, n, k, group, torch.float16)
    wide_codes = torch.full((n, k // 2 + 5), 0xff, device="cuda", dtype=torch.uint8)
    wide_scales = torch.full((n, 13, 2), float("nan"), device="cuda", dtype=torch.float16)
    wide_codes[:, 3:3 + k // 2], wide_scales[:, 2:11] = packed_pairs(codes), scales
    packed = torch.empty(bd.w4_bytes(n, k, group), device="cuda", dtype=torch.uint8)
    bd.w4_pack(wide_codes[:, 3:3 + k // 2], wide_scales[:, 2:11], packed, group=group)
    assert (packed == pack(bd, codes, scales, group)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_steps_of_zero_negative_steps_and_every_code(bd, dtype):
    """Pairs are what the caller gives: any sign; a group of one value has step 0."""
    n, k, group = 32, 256, 32
    codes = (torch.arange(n * k, device="cuda") * 7 % 16).view(n, k).double()
    scales = torch.stack([randn(1, n, 8, dtype=dtype), randn(2, n, 8, dtype=dtype)], -1)
    scales[:, 3, 0] = 0
    packed = pack(bd, codes, scales, group)
    for m in (1, 20):
        x = randn(3, m, k, dtype=dtype)
        check(run(bd, x, packed, n, group), x, codes, scales, group)


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e-12), (torch.bfloat16, 1e15), (torch.float16, 2.0 ** -18), (torch.float16, 1e4)])
def test_magnitudes(bd, dtype, size):
    n, k, group = 64, 512, 32
    codes, scales = weights(8, n, k, group, dtype)
    if dtype == torch.float16 and size > 1:
        scales = scales / 64                  # (the sums stay in FP16)
    packed = pack(bd, codes, scales, group)
    for m in (1, 12):
        x = randn(9, m, k, dtype=torch.float32, scale=size).to(dtype)
        check(run(bd, x, packed, n, group), x, codes, scales, group)


def test_values_that_are_not_finite_stay_in_their_rows_and_columns(bd):
    n, k, group = 48, 256, 64
    codes, scales = weights(10, n, k, group, torch.bfloat16)
    scales[20, 1, 0] = float("nan")
    scales[30, 2, 1] = float("inf")
    packed = pack(bd, codes, scales, group)
    x = randn(11, 5, k)
    x[2, 100] = float("nan")
    x[4, 200] = float("inf")
    y = run(bd, x, packed, n, group)
    assert not torch.isfinite(y[[2, 4]]).any() and not torch.isfinite(y[:, [20, 30]]).any()
    rows, cols = [0, 1, 3], [c for c in range(n) if c not in (20, 30)]
    check(y[rows][:, cols], x[rows], codes[cols], scales[cols], group)


def test_no_rows_streams_repeats_and_capture(bd):
    n, k, group = 1000, 1280, 128
    codes, scales = weights(12, n, k, group, torch.bfloat16)
    packed = pack(bd, codes, scales, group)
    run(bd, torch.empty(0, k, device="cuda", dtype=torch.bfloat16), packed, n, group)
    x = randn(13, 9, k)
    want = run(bd, x, packed, n, group)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    y = run(bd, x, packed, n, group, stream=side)
    side.synchronize()
    assert (y == want).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bd.linear_w4_fwd(x, packed, None, y, group=group)
    x.copy_(randn(14, 9, k))
    g.replay()
    torch.cuda.synchronize()
    check(y, x, codes, scales, group)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 8), (16, 128), (17, 136), (100, 648), (1291, 1368), (33, 10240)])
def test_the_matrix_back_in_16_bits(bd, n, k, group, dtype):
    """Bit for bit: each value rounded once, to the largest finite one where it lies beyond; what is not the matrix's is left."""
    codes, scales = weights(n + k, n, k, group, dtype)
    most = torch.finfo(dtype).max
    scales[0, 0, 0], scales[0, 0, 1] = most / 8, most / 2
    codes[0, :8] = torch.arange(8, 16, device="cuda")
    if n > 1:
        scales[1, 0] = float("nan")
    wide = torch.full((n + 2, k + 16), 7.0, device="cuda", dtype=dtype)
    bd.w4_unpack(pack(bd, codes, scales, group), wide[1:n + 1, 8:k + 8], group=group)
    got, want = wide[1:n + 1, 8:k + 8].clone(), values(codes, scales, group).clamp(-most, most).to(dtype)
    assert ((got == want) | (torch.isnan(got) & torch.isnan(want))).all()
    assert int(torch.isnan(got).sum()) == (min(group, k) if n > 1 else 0)
    wide[1:n + 1, 8:k + 8] = 7.0
    assert (wide == 7.0).all() and bd.device_status() == 0


def test_refusals_of_the_matrix_back(bd):
    codes, scales = weights(3, 20, 128, 32, torch.bfloat16)
    packed, w = pack(bd, codes, scales, 32), torch.zeros(20, 128, device="cuda", dtype=torch.bfloat16)
    for call in (lambda: bd.w4_unpack(packed[:-1], w, group=32), lambda: bd.w4_unpack(packed, w, group=64), lambda: bd.w4_unpack(packed, w, group=16),
                 lambda: bd.w4_unpack(packed, w.repeat(1, 2), group=32), lambda: bd.w4_unpack(packed, w.float(), group=32),
                 lambda: bd.w4_unpack(packed, w[:1].expand(20, 128), group=32), lambda: bd.w4_unpack(packed, w.t().contiguous().t(), group=32),
                 lambda: bd.w4_unpack(packed.view(torch.int8), w, group=32), lambda: bd.w4_unpack(packed, w.cpu(), group=32)):
        with pytest.raises(bd.BdattnError):
            call()
    L = bd.lib()
    good = dict(packed=packed.data_ptr(), w=w.data_ptr(), ld=128, N=20, K=128, group=32, dtype=bd.BF16)
    for field, value, reason in (("packed", 0, "null"), ("w", 0, "null"), ("w", w.data_ptr() + 8, "aligned"), ("ld", 120, "row stride"), ("ld", 132, "multiple of 8"),
                                 ("N", 0, "N must"), ("K", 132, "multiple of 8"), ("K", (1 << 30) + 8, "2^30"), ("group", 48, "group"), ("dtype", bd.F32, "dtype")):
        c = dict(good, **{field: value})
        assert L.bdattn_w4_unpack(c["packed"], c["w"], c["ld"], c["N"], c["K"], c["group"], c["dtype"], None) == -1
        assert reason in bd.last_error(), (field, bd.last_error())
    assert (w == 0).all()


def test_refusals(bd):
    n, k, group = 32, 128, 32
    codes, scales = weights(15, n, k, group, torch.bfloat16)
    pairs, packed = packed_pairs(codes), pack(bd, codes, scales, group)
    x, y = randn(1, 3, k), torch.empty(3, n, device="cuda", dtype=torch.bfloat16)
    for call in (lambda: bd.linear_w4_fwd(x, packed, None, y, group=64),                    # bytes of another packing
                 lambda: bd.linear_w4_fwd(x, packed, None, y, group=48),
                 lambda: bd.linear_w4_fwd(x, packed[:-16], None, y, group=group),
                 lambda: bd.linear_w4_fwd(x, packed.view(torch.int8), None, y, group=group),
                 lambda: bd.linear_w4_fwd(x.half(), packed, None, y, group=group),
                 lambda: bd.linear_w4_fwd(x.float(), packed, None, y.float(), group=group),
                 lambda: bd.linear_w4_fwd(x[:2], packed, None, y, group=group),
                 lambda: bd.linear_w4_fwd(x, packed, y[0].half(), y, group=group),
                 lambda: bd.linear_w4_fwd(x, packed, y[0, :31], y, group=group),
                 lambda: bd.linear_w4_fwd(x, packed, None, y, group=group, gate=y[0].float()),
                 lambda: bd.linear_w4_fwd(x, packed, None, y, group=group, residual=y[:2]),
                 lambda: bd.linear_w4_fwd(x, packed, None, y, group=group, act="relu"),
                 lambda: bd.linear_w4_fwd(randn(1, 3, 132)[:, 4:], packed, None, y, group=group),       # rows off 16 bytes
                 lambda: bd.w4_pack(pairs, scales, packed[:-1], group=group),
                 lambda: bd.w4_pack(pairs, scales[:, :3], packed, group=group),
                 lambda: bd.w4_pack(pairs, scales.float(), packed, group=group),
                 lambda: bd.w4_pack(pairs[:, :62], scales, packed, group=group),
                 lambda: bd.w4_pack(pairs.view(torch.int8), scales, packed, group=group),
                 lambda: bd.w4_pack(pairs, scales, packed, group=16)):
        with pytest.raises(bd.BdattnError):
            call()
    assert bd.w4_bytes(0, 8, 32) == bd.w4_bytes(8, 0, 32) == bd.w4_bytes(8, 8, 33) == 0
    p = bd.LinearW4Params(dtype=bd.BF16, M=3, N=n, K=k, group=group, x=x.data_ptr(), w=packed.data_ptr(), y=y.data_ptr(), act=9)
    for field, value, reason in (("act", 9, "activation"), ("K", 132, "multiple of 8"), ("x_ld", 132, "multiple of 8"), ("x", 0, "null"),
                                 ("y_ld", 8, "row stride"), ("w", packed.data_ptr() + 8, "aligned"), ("M", 600000, "rows"), ("K", (1 << 30) + 8, "2^30"), ("M", -1, ">= 0")):
        q = bd.LinearW4Params.from_buffer_copy(p)
        q.act = 0
        setattr(q, field, value)
        assert bd.lib().bdattn_linear_w4_fwd(q, None) == -1 and reason in bd.last_error(), field
