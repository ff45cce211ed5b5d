"""The norms behind one block and ahead of the next against their formulas in 64 bits.

Tolerances.  Units of rounding: u = 2^-8 (BF16), 2^-11 (FP16), 2^-4 (e4m3, and half of its smallest step, 2^-10, below
2^-6).  The FP32 part: two sums of n squares in at most n / 32 + 50 steps of 2^-24 and two approximate roots of 2^-22, below
1e-5 relative for these widths.  h is a sum whose terms may cancel: its FP32 error is 1e-5 of |residual_scale r| + |gate b|,
and that of y the same multiplied by gain / rms(h)."""
import pytest
import torch

from four_bit import UNIT, randn

pytestmark = pytest.mark.gpu

F32_PART = 1e-5
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}       # half of the smallest step
E4M3 = torch.float8_e4m3fn


def formula(x, r, post, gate, scale, gain, eps):
    """h, y, and what their FP32 error is in proportion to"""
    b = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + eps)
    if post is not None:
        b = b * post.double()
    if gate is not None:
        gate = gate.reshape(-1, x.shape[1])
        b = b * gate.double().repeat_interleave(len(x) // len(gate), 0)
    h, size = scale * r.double() + b, (scale * r.double()).abs() + b.abs()
    f = 1 / torch.sqrt(h.square().mean(1, keepdim=True) + eps)
    if gain is not None:
        f = f * gain.double()
    return h, h * f, size, size * f.abs()


def call(bd, x, r, post=None, gate=None, scale=1.0, gain=None, out_dtype=None, eps=1e-6, **kw):
    out = torch.full(x.shape, 3.0, device="cuda").to(out_dtype) if out_dtype is not None else None
    out_scale = torch.full((x.shape[0],), float("nan"), device="cuda") if out_dtype == E4M3 else None
    h = torch.full_like(x, float("nan"))
    bd.sandwich_norm_fwd(x, r, h, post, gate=gate, residual_scale=scale, gain=gain, out=out, out_scale=out_scale, eps=eps, **kw)
    assert bd.device_status() == 0
    return h, out, out_scale


def check(got, x, r, post=None, gate=None, scale=1.0, gain=None, eps=1e-6):
    h, out, out_scale = got
    h_ref, y, h_size, y_size = formula(x, r, post, gate, scale, gain, eps)
    u = UNIT[x.dtype]
    err = (h.double() - h_ref).abs()
    assert (err <= u * h_ref.abs() + F32_PART * h_size + TINY[x.dtype]).all(), float((err / h_size).max())
    if out is None:
        return
    if out_scale is None:
        err = (out.double() - y).abs()
        assert (err <= u * y.abs() + F32_PART * y_size + TINY[x.dtype]).all(), float((err / y_size).max())
        return
    top = y.abs().amax(1)
    assert ((out_scale.double() * 448 - top).abs() <= 2 * F32_PART * y_size.amax(1) + 1e-35).all()
    s = out_scale.double()[:, None]
    err = (out.double() * s - y).abs()
    assert (err <= 2.0 ** -4 * y.abs() + 3 * F32_PART * y_size.amax(1, keepdim=True) + s * 2.0 ** -10).all(), float(err.max())
    assert (err.square().mean().sqrt() <= 2.0 ** -4 / 3 ** 0.5 * y.square().mean().sqrt() + s.max() * 2.0 ** -10).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["none", "same", "fp8"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (2, 33), (17, 64), (5, 256), (1, 2560), (129, 264), (37, 1365), (64, 1288),
                                       (7, 5120), (300, 640), (300, 1024), (200, 4096), (2, 8192), (3, 8200), (2, 16370), (2, 16376), (1, 40961)])
def test_against_the_formula(bd, rows, cols, kind, dtype):
    x, r = randn(rows + cols, rows, cols, dtype=dtype), randn(rows + cols + 1, rows, cols, dtype=dtype, scale=2.0)
    post, gain = (1 + randn(cols + i, cols, dtype=dtype, scale=0.02) for i in (1, 2))
    gate = randn(cols + 3, cols, dtype=dtype, scale=0.5)
    out = {"none": None, "same": dtype, "fp8": E4M3}[kind]
    gain = gain if out is not None else None
    check(call(bd, x, r, post, gate, 0.7, gain, out), x, r, post, gate, 0.7, gain)
    check(call(bd, x, r, None, None, 1.0, None, out), x, r)


@pytest.mark.parametrize("rows", [1, 147, 149, 600, 5000])
@pytest.mark.parametrize("cols", [64, 200, 320, 2048])
def test_many_rows(bd, rows, cols):
    x, r = randn(rows, rows, cols), randn(rows + 1, rows, cols)
    for out in (None, torch.bfloat16, E4M3):
        check(call(bd, x, r, out_dtype=out), x, r)


@pytest.mark.parametrize("cols", [640, 645, 20000])
@pytest.mark.parametrize("gates", [1, 2, 3, 12])
def test_a_gate_for_each_group_of_rows(bd, gates, cols):
    x, r = randn(1, 12, cols), randn(2, 12, cols)
    wide = randn(3, gates, cols + 24, scale=0.5)
    for gate in (wide[:, :cols], wide[:, :cols].contiguous(), wide[:, 3:3 + cols]):
        check(call(bd, x, r, None, gate, 1.0, None, torch.bfloat16), x, r, None, gate)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_gains(bd, dtype):
    x, r = randn(1, 9, 1280, dtype=torch.float16), randn(2, 9, 1280, dtype=torch.float16)
    g = [randn(3 + i, 1280, dtype=dtype) for i in range(2)]
    for post in (None, g[0]):
        for gain in (None, g[1]):
            check(call(bd, x, r, post, None, 1.0, gain, torch.float16), x, r, post, None, 1.0, gain)


@pytest.mark.parametrize("scale", [0.0, -1.5, 1e-3, 300.0])
def test_the_streams_scale(bd, scale):
    x, r = randn(1, 9, 1280), randn(2, 9, 1280)
    check(call(bd, x, r, scale=scale, out_dtype=torch.bfloat16), x, r, scale=scale)


@pytest.mark.parametrize("cols", [520, 519])
@pytest.mark.parametrize("skip", [0, 1, 4, 8])
@pytest.mark.parametrize("width", [528, 533, 536])
def test_rows_inside_wider_tensors(bd, cols, skip, width):
    """Any stride and alignment, and nothing written beside the rows."""
    if skip + cols > width:
        pytest.skip("does not fit")
    rows = 21
    for out_dtype in (torch.bfloat16, E4M3):
        wide = [randn(i, rows, width) for i in range(2)] + [torch.full((rows, width), 7.0, device="cuda", dtype=torch.bfloat16),
                                                            torch.full((rows, width), 7.0, device="cuda").to(out_dtype)]
        x, r, h, out = [w[:, skip:skip + cols] for w in wide]
        scale = torch.empty(rows, device="cuda") if out_dtype == E4M3 else None
        before = [w.clone() for w in wide]
        bd.sandwich_norm_fwd(x, r, h, out=out, out_scale=scale)
        check((h, out, scale), x, r)
        for w, b in zip(wide[2:], before[2:]):
            kept = torch.ones(width, dtype=torch.bool)
            kept[skip:skip + cols] = False
            assert (w.view(torch.uint8).view(rows, width, -1)[:, kept] == b.view(torch.uint8).view(rows, width, -1)[:, kept]).all()


def test_tensors_that_are_off_by_different_amounts(bd):
    x, r = randn(1, 6, 641)[:, 1:], randn(2, 6, 643)[:, 3:]
    h, out = torch.empty(6, 640, device="cuda", dtype=torch.bfloat16), torch.empty(6, 642, device="cuda", dtype=torch.bfloat16)[:, 2:]
    bd.sandwich_norm_fwd(x, r, h, out=out)
    check((h, out, None), x, r)


@pytest.mark.parametrize("cols", [640, 333, 20000])
def test_outputs_in_the_place_of_inputs(bd, cols):
    x, r = randn(5, 12, cols), randn(6, 12, cols)
    want = call(bd, x, r, out_dtype=torch.bfloat16)
    x1, r1 = x.clone(), r.clone()
    bd.sandwich_norm_fwd(x1, r1, r1, out=x1)                   # the stream updated, the rows in the place of the branch
    assert (r1 == want[0]).all() and (x1 == want[1]).all()
    x2, r2, out = x.clone(), r.clone(), torch.empty_like(x)
    bd.sandwich_norm_fwd(x2, r2, x2, out=out)
    assert (x2 == want[0]).all() and (out == want[1]).all() and (r2 == r).all()


@pytest.mark.parametrize("cols", [256, 255, 2560, 20000])
def test_rows_of_zeros_and_values_that_are_not_finite(bd, cols):
    x, r = randn(3, 7, cols), randn(4, 7, cols)
    x[1], r[1] = 0, 0
    x[2] = 0
    x[3, 5], x[4, 7], r[5, 9] = float("inf"), float("nan"), float("nan")
    fine = [0, 1, 2, 6]
    h, out, _ = call(bd, x, r, out_dtype=torch.bfloat16)
    check((h[fine], out[fine], None), x[fine], r[fine])
    assert torch.isnan(h[3:5]).all() and torch.isnan(out[3:6]).all() and int(torch.isnan(h[5]).sum()) == 1
    h, q, scale = call(bd, x, r, out_dtype=E4M3)
    check((h[fine], q[fine], scale[fine]), x[fine], r[fine])
    assert torch.isnan(scale[3:6]).all() and scale[1] == 0 and (q[1].float() == 0).all()


@pytest.mark.parametrize("eps", [0.0, 1e-6, 1.0])
@pytest.mark.parametrize("size", [1e-3, 1.0, 1e3])
def test_epsilon_and_magnitudes(bd, eps, size):
    x, r = randn(8, 4, 2048, scale=size), randn(9, 4, 2048, scale=size)
    for out in (torch.bfloat16, E4M3):
        check(call(bd, x, r, eps=eps, out_dtype=out), x, r, eps=eps)


def test_rows_of_zeros_without_an_epsilon(bd):
    x, r = randn(1, 3, 640), randn(2, 3, 640)
    x[1], x[2], r[2] = 0, 0, 0
    for cols in (640, 333):
        h, out, _ = call(bd, x[:, :cols], r[:, :cols], eps=0.0, out_dtype=torch.bfloat16)
        assert (h[1] == r[1, :cols]).all() and (h[2] == 0).all() and (out[2] == 0).all() and torch.isfinite(out).all()
        h, q, scale = call(bd, x[:, :cols], r[:, :cols], eps=0.0, out_dtype=E4M3)
        assert scale[2] == 0 and (q[2].float() == 0).all() and torch.isfinite(scale).all()


def test_no_rows_streams_and_repeats(bd):
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    bd.sandwich_norm_fwd(x, torch.empty_like(x), torch.empty_like(x), out=torch.empty_like(x))
    x, r = randn(9, 500, 1024), randn(10, 500, 1024)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    a = call(bd, x, r, out_dtype=E4M3, stream=side)
    side.synchronize()
    check(a, x, r)
    b = call(bd, x, r, out_dtype=E4M3)
    for p, q in zip(a, b):
        assert (p.view(torch.uint8) == q.view(torch.uint8)).all()


def test_graph_capture(bd):
    x, r = randn(12, 16, 2560), randn(13, 16, 2560)
    out, h = torch.empty_like(x), torch.empty_like(x)
    bd.sandwich_norm_fwd(x, r, h, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bd.sandwich_norm_fwd(x, r, h, out=out)
    x.copy_(randn(14, 16, 2560))
    g.replay()
    torch.cuda.synchronize()
    check((h, out, None), x, r)


def test_refusals(bd):
    x = randn(1, 4, 64)
    h, q, s = torch.empty_like(x), torch.empty(4, 64, device="cuda", dtype=E4M3), torch.empty(4, device="cuda")
    gate = randn(2, 2, 64)
    for call_ in (lambda: bd.sandwich_norm_fwd(x, x, h, out=q),                                 # no scales
                  lambda: bd.sandwich_norm_fwd(x, x, h, out=h, out_scale=s),                    # scales of nothing
                  lambda: bd.sandwich_norm_fwd(x, x, h, out_scale=s),
                  lambda: bd.sandwich_norm_fwd(x, x, h, gain=gate[0]),                          # a gain without an output
                  lambda: bd.sandwich_norm_fwd(x, x, h, out=x.half()),
                  lambda: bd.sandwich_norm_fwd(x, x.half(), h),
                  lambda: bd.sandwich_norm_fwd(x, x, h.half()),
                  lambda: bd.sandwich_norm_fwd(x.float(), x.float(), h.float()),
                  lambda: bd.sandwich_norm_fwd(x, x[:2], h),
                  lambda: bd.sandwich_norm_fwd(x, x, h, gate[0].half()),
                  lambda: bd.sandwich_norm_fwd(x, x, h, gate[0], gain=gate[0].float(), out=q, out_scale=s),      # two types
                  lambda: bd.sandwich_norm_fwd(x, x, h, s),
                  lambda: bd.sandwich_norm_fwd(x, x, h, gate=gate.float()),
                  lambda: bd.sandwich_norm_fwd(x, x, h, gate=randn(3, 3, 64)),                  # 3 does not divide 4
                  lambda: bd.sandwich_norm_fwd(x, x, h, gate=gate[:, :32]),
                  lambda: bd.sandwich_norm_fwd(x, x, h, gate=gate[:0]),
                  lambda: bd.sandwich_norm_fwd(x, x, h, out=q, out_scale=s[:3]),
                  lambda: bd.sandwich_norm_fwd(x.t(), x.t(), h.t()),
                  lambda: bd.sandwich_norm_fwd(x, x, h, residual_scale=float("nan")),
                  lambda: bd.sandwich_norm_fwd(x, x, h, residual_scale=float("inf")),
                  lambda: bd.sandwich_norm_fwd(x, x, h, eps=-1.0)):
        with pytest.raises(bd.BdattnError):
            call_()
    p = bd.SandwichNormParams(dtype=bd.BF16, rows=4, cols=64, x=x.data_ptr(), residual=x.data_ptr(), residual_out=h.data_ptr(), x_ld=32)
    assert bd.lib().bdattn_sandwich_norm_fwd(p, None) == -1 and "row stride" in bd.last_error()
    p.x_ld, p.x = 0, x.data_ptr() + 1
    assert bd.lib().bdattn_sandwich_norm_fwd(p, None) == -1 and "aligned" in bd.last_error()
    p.x = 0
    assert bd.lib().bdattn_sandwich_norm_fwd(p, None) == -1 and "null" in bd.last_error()
    assert bd.lib().bdattn_sandwich_norm_fwd(None, None) == -1
