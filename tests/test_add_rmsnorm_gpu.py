"""Residual addition + RMSNorm, 16-bit and e4m3 outputs, against the formulas in 64 bits.

Tolerances.  Units of rounding: u = 2^-8 (BF16), 2^-11 (FP16), 2^-4 (e4m3, and half of its smallest step, 2^-10,
below 2^-6).  The FP32 part: a sum of n squares in at most n / 32 + 50 steps of 2^-24, an approximate
root and reciprocal of 2^-22 each, a few products: below 1e-5 relative for the widths used here."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32_PART = 1e-5
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}       # half of the smallest step
E4M3 = torch.float8_e4m3fn


def randn(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


def formula(x, residual, gain, eps):
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return h, y if gain is None else y * gain.double()


def run(bd, x, gain, residual, out_dtype, eps=1e-6, residual_out="new", **kw):
    out = torch.full(x.shape, 3.0, device="cuda").to(out_dtype)
    scale = torch.full((x.shape[0],), float("nan"), device="cuda") if out_dtype == E4M3 else None
    if residual_out == "new":
        residual_out = torch.full_like(x, float("nan")) if residual is not None else None
    bd.add_rmsnorm_fwd(x, out, gain, residual=residual, residual_out=residual_out, out_scale=scale, eps=eps, **kw)
    assert bd.device_status() == 0
    return out, scale, residual_out


def near(got, ref, unit, tiny, what):
    err = (got.double() - ref).abs()
    bad = err > (unit + F32_PART) * ref.abs() + tiny
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float((err / ref.abs().clamp_min(1e-30)).max()):.3g}"


def check(out, scale, residual_out, x, residual, gain, eps=1e-6):
    h, y = formula(x, residual, gain, eps)
    if residual_out is not None:
        near(residual_out, h, UNIT[x.dtype] * (1 + 2.0 ** -12), TINY[x.dtype], "residual_out")
    if scale is None:
        near(out, y, UNIT[x.dtype], TINY[x.dtype], "out")
        return
    near(scale, y.abs().amax(1) / 448, 0.0, 1e-37, "out_scale")
    s = scale.double()[:, None]
    err = (out.double() * s - y).abs()
    assert (err <= (2.0 ** -4 + 2 * F32_PART) * y.abs() + s * (2.0 ** -10 + 1e-4)).all(), float(err.max())
    # rounded to the nearest, no further step away: the root mean square of the error is that of a uniform
    # distribution over a step, at most 2^-4 / sqrt(3) of the value
    assert (err.square().mean().sqrt() <= 2.0 ** -4 / 3 ** 0.5 * y.square().mean().sqrt() + s.max() * 2.0 ** -10).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (2, 33), (5, 256), (1, 2560), (129, 264), (37, 1365), (64, 1288),
                                       (7, 5120), (300, 640), (2, 8192), (3, 8200), (2, 20000), (2, 32776), (1, 40961), (1, 70000)])
def test_against_the_formula(bd, rows, cols, fp8, dtype):
    x, r = randn(rows + cols, rows, cols, dtype=dtype), randn(rows + cols + 1, rows, cols, dtype=dtype, scale=2.0)
    g = 1 + randn(cols, cols, dtype=dtype, scale=0.02)
    for residual in (None, r):
        got = run(bd, x, g, residual, E4M3 if fp8 else dtype)
        check(*got, x, residual, g)


@pytest.mark.parametrize("rows", [1, 147, 149, 600, 5000])
@pytest.mark.parametrize("cols", [64, 320, 2048])
def test_many_rows(bd, rows, cols):
    x, r = randn(rows, rows, cols), randn(rows + 1, rows, cols)
    check(*run(bd, x, None, r, torch.bfloat16), x, r, None)
    check(*run(bd, x, None, r, E4M3), x, r, None)


@pytest.mark.parametrize("gain_dtype", [None, torch.float32, torch.float16])
def test_gains(bd, gain_dtype):
    x = randn(1, 9, 1280, dtype=torch.float16)
    g = None if gain_dtype is None else randn(2, 1280, dtype=gain_dtype)
    check(*run(bd, x, g, None, torch.float16), x, None, g)
    check(*run(bd, x, g, None, E4M3), x, None, g)


@pytest.mark.parametrize("cols", [520, 519])
@pytest.mark.parametrize("skip", [0, 1, 4, 8])
@pytest.mark.parametrize("width", [528, 533, 536])
def test_rows_inside_wider_tensors(bd, cols, skip, width):
    """Any stride and alignment, and nothing written beside the rows."""
    rows = 21
    for out_dtype in (torch.bfloat16, E4M3):
        wide = [randn(i, rows, width) for i in range(2)] + [torch.full((rows, width), 7.0, device="cuda", dtype=torch.bfloat16),
                                                            torch.full((rows, width), 7.0, device="cuda").to(out_dtype)]
        cut = [w[:, skip:skip + cols] for w in wide] if skip + cols <= width else None
        if cut is None:
            pytest.skip("does not fit")
        x, r, ro, out = cut
        scale = torch.empty(rows, device="cuda") if out_dtype == E4M3 else None
        before = [w.clone() for w in wide]
        bd.add_rmsnorm_fwd(x, out, None, residual=r, residual_out=ro, out_scale=scale)
        check(out, scale, ro, x, r, None)
        for w, b in zip(wide[2:], before[2:]):
            kept = torch.ones(width, dtype=torch.bool)
            kept[skip:skip + cols] = False
            assert (w.view(torch.uint8).view(rows, width, -1)[:, kept] == b.view(torch.uint8).view(rows, width, -1)[:, kept]).all()


@pytest.mark.parametrize("cols", [640, 333, 33000])
def test_outputs_in_the_place_of_inputs(bd, cols):
    x, r = randn(5, 12, cols), randn(6, 12, cols)
    want = run(bd, x, None, r, torch.bfloat16)
    x1, r1 = x.clone(), r.clone()
    bd.add_rmsnorm_fwd(x1, x1, None, residual=r1, residual_out=r1)            # the stream and the rows updated in place
    assert (x1 == want[0]).all() and (r1 == want[2]).all()
    x2, r2, out = x.clone(), r.clone(), torch.empty_like(x)
    bd.add_rmsnorm_fwd(x2, out, None, residual=r2, residual_out=x2)
    assert (out == want[0]).all() and (x2 == want[2]).all() and (r2 == r).all()


def test_rows_of_zeros_and_values_that_are_not_finite(bd):
    for cols in (256, 255):
        x = randn(3, 6, cols)
        x[1] = 0
        x[3, 5] = float("inf")
        x[4, 7] = float("nan")
        out, _, _ = run(bd, x, None, None, torch.bfloat16)
        q, scale, _ = run(bd, x, None, None, E4M3)
        fine = [0, 1, 2, 5]
        check(out[fine], None, None, x[fine], None, None)
        check(q[fine], scale[fine], None, x[fine], None, None)
        assert (out[1] == 0).all() and scale[1] == 0 and (q[1].float() == 0).all()
        assert torch.isnan(out[3, 5]) and torch.isnan(out[4]).all() and torch.isnan(scale[3:5]).all()


@pytest.mark.parametrize("eps", [0.0, 1e-6, 1.0])
@pytest.mark.parametrize("size", [1e-3, 1.0, 1e3])
def test_epsilon_and_magnitudes(bd, eps, size):
    x = randn(8, 4, 2048, scale=size)
    check(*run(bd, x, None, None, torch.bfloat16, eps=eps), x, None, None, eps)
    check(*run(bd, x, None, None, E4M3, eps=eps), x, None, None, eps)


def test_no_rows_and_other_streams(bd):
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    bd.add_rmsnorm_fwd(x, torch.empty_like(x))
    side = torch.cuda.Stream()
    x = randn(9, 500, 1024)
    torch.cuda.synchronize()
    out = torch.empty_like(x)
    bd.add_rmsnorm_fwd(x, out, stream=side)
    with torch.cuda.stream(side):
        out2 = torch.empty_like(x)
        bd.add_rmsnorm_fwd(out, out2)           # ordered behind the first by the stream alone
    side.synchronize()
    check(out, None, None, x, None, None)
    check(out2, None, None, out, None, None)


def test_the_same_call_gives_the_same_bits(bd):
    x, r = randn(10, 700, 1536), randn(11, 700, 1536)
    a, b = (run(bd, x, None, r, E4M3) for _ in range(2))
    for p, q in zip(a, b):
        assert (p.view(torch.uint8) == q.view(torch.uint8)).all()


def test_graph_capture(bd):
    x, r = randn(12, 16, 2560), randn(13, 16, 2560)
    out, ro = torch.empty_like(x), torch.empty_like(x)
    bd.add_rmsnorm_fwd(x, out, None, residual=r, residual_out=ro)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bd.add_rmsnorm_fwd(x, out, None, residual=r, residual_out=ro)
    x.copy_(randn(14, 16, 2560))
    g.replay()
    torch.cuda.synchronize()
    check(out, None, ro, x, r, None)


def test_refusals(bd):
    x = randn(1, 4, 64)
    out, q, s = torch.empty_like(x), torch.empty(4, 64, device="cuda", dtype=E4M3), torch.empty(4, device="cuda")
    E = bd.BdattnError
    for call in (lambda: bd.add_rmsnorm_fwd(x, q),                                                  # no scales
                 lambda: bd.add_rmsnorm_fwd(x, out, out_scale=s),                                   # scales of nothing
                 lambda: bd.add_rmsnorm_fwd(x, out.half()),                                         # another 16-bit type
                 lambda: bd.add_rmsnorm_fwd(x.float(), out),
                 lambda: bd.add_rmsnorm_fwd(x, torch.empty(4, 32, device="cuda", dtype=x.dtype)),
                 lambda: bd.add_rmsnorm_fwd(x, out, residual=x[:2]),
                 lambda: bd.add_rmsnorm_fwd(x, out, residual=x.half()),
                 lambda: bd.add_rmsnorm_fwd(x, out, residual_out=x.half()),
                 lambda: bd.add_rmsnorm_fwd(x, out, s),                                             # gain of another length
                 lambda: bd.add_rmsnorm_fwd(x, out, torch.ones(64, device="cuda").half()),          # gain of another type
                 lambda: bd.add_rmsnorm_fwd(x, q, out_scale=s.double()),
                 lambda: bd.add_rmsnorm_fwd(x, q, out_scale=s[:3]),
                 lambda: bd.add_rmsnorm_fwd(x.t(), out.t()),
                 lambda: bd.add_rmsnorm_fwd(x[0], out[0]),
                 lambda: bd.add_rmsnorm_fwd(x, out, eps=-1.0),
                 lambda: bd.add_rmsnorm_fwd(x, out, eps=float("nan"))):
        with pytest.raises(E):
            call()
    p = bd.AddRmsNormParams(dtype=bd.BF16, rows=4, cols=64, x=x.data_ptr(), out=out.data_ptr(), out_dtype=bd.BF16, x_ld=32)
    assert bd.lib().bdattn_add_rmsnorm_fwd(p, None) == -1 and "row stride" in bd.last_error()
    p.x_ld, p.x = 0, x.data_ptr() + 1
    assert bd.lib().bdattn_add_rmsnorm_fwd(p, None) == -1 and "aligned" in bd.last_error()
    p.x, p.rows = 0, 4
    assert bd.lib().bdattn_add_rmsnorm_fwd(p, None) == -1 and "null" in bd.last_error()
    assert bd.lib().bdattn_add_rmsnorm_fwd(None, None) == -1
    assert (x == randn(1, 4, 64)).all()
