"""A layer's operators at the ends of the range of their types, against their formulas in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


# Kernels: few rows, a tile over a cluster, single tiles, pairs (tests/layer_shapes.py).
@pytest.mark.parametrize("M,N,K", [(2, 64, 64), (12, 64, 64), (17, 64, 1280), (129, 1288, 648), (900, 2432, 648)])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("fp8", [False, True])
def test_activations_of_large_sums(bd, M, N, K, act, fp8):
    """act(z) of a large negative z is 0 and of a large positive one z, up to the largest sums that FP32 holds."""
    K = K // 16 * 16
    z = torch.tensor([-3e38, -1e38, -1e37, -3e35, -1e30, -1e20, -1e9, -1e4, -200.0, -100.0, -89.0, -88.0, -87.0, -20.0, -12.0, -10.0, -9.0,
                      0.0, 9.0, 12.0, 88.0, 200.0, 1e4, 1e20, 1e30, 3e38], device="cuda").to(BF16)
    bias = z[torch.arange(N, device="cuda") % len(z)].contiguous()
    x = torch.zeros(M, K, device="cuda", dtype=BF16)
    w = torch.zeros(N, K, device="cuda", dtype=BF16)
    if fp8:
        x, w = x.to(E4M3), w.to(E4M3)
    y = torch.full((M, N), 7.0, device="cuda", dtype=BF16)
    bd.linear_act_fwd(x, w, bias, y, act=act)
    b = bias.double()
    u = {"silu": b, "gelu": b, "gelu_tanh": 2 * (2 / torch.pi) ** 0.5 * (b + 0.044715 * b ** 3)}[act]
    ref = b * (torch.special.ndtr(b) if act == "gelu" else torch.sigmoid(u))
    # the output's rounding, the activation's own error (4e-6 |z| where its slope is not flat, which it is below -20), and
    # values below the smallest normal of BF16 and FP32
    bound = 2.0 ** -8 * ref.abs() + torch.where(b < -20, 0.0, 4e-6 * b.abs()) + 1e-8 * (b >= -100) + 1e-30
    assert ((y.double() - ref).abs() <= bound).all(), (y.double() - ref).abs().amax(0)
    nan = torch.full((N,), float("nan"), device="cuda", dtype=BF16)
    bd.linear_act_fwd(x, w, nan, y, act=act)
    assert torch.isnan(y).all()


def norm(bd, x, residual=None, gain=None, eps=1e-6, skip=0):
    """(values of 8 bits times their scale, scale, values); skip: elements that the rows lie off 16 bytes."""
    rows, cols = x.shape
    wide = lambda t: torch.nn.functional.pad(t, (skip, 8 - skip)) if skip else t
    cut = lambda t: t[:, skip:skip + cols]
    q = cut(wide(torch.zeros(rows, cols, device="cuda")).to(E4M3))
    scale = torch.full((rows,), 7.0, device="cuda")
    bd.add_rmsnorm_fwd(cut(wide(x)), q, gain, residual=None if residual is None else cut(wide(residual)), out_scale=scale, eps=eps)
    return q.double() * scale.double()[:, None], scale, q


# Kernels: a row to eight lanes, to a warp, to a CTA, wide rows read twice; rows off 16 bytes; tensors off by different numbers
# of elements (the last column count)
WIDTHS = [(4, 64, 0), (4, 512, 0), (200, 1024, 0), (3, 5120, 0), (300, 6000, 0), (2, 20000, 0), (4, 519, 3), (300, 5001, 3), (2, 20001, 5)]


@pytest.mark.parametrize("rows,cols,skip", WIDTHS)
@pytest.mark.parametrize("off", [False, True])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("gain", [0.0, 1.0])
def test_rows_with_a_value_that_is_not_finite_have_scale_nan(bd, rows, cols, skip, off, value, gain):
    """Whatever gain stands at the value's column."""
    x = torch.ones(rows, cols, device="cuda", dtype=BF16)
    for i, c in enumerate((0, cols // 2, cols - 1)):
        x[i % rows, c] = value
    bad = ~torch.isfinite(x).all(1)
    w = torch.ones(cols, device="cuda", dtype=BF16)
    w[[0, cols // 2, cols - 1]] = gain
    r = torch.zeros(rows, cols + 5, device="cuda", dtype=BF16)[:, 5:] if off else None
    got, scale, q = norm(bd, x, r, w, skip=skip)
    assert torch.isnan(scale[bad]).all() and ((scale[~bad] * 448 - 1).abs() < 1e-5).all()


@pytest.mark.parametrize("rows,cols,skip", WIDTHS)
@pytest.mark.parametrize("off", [False, True])
@pytest.mark.parametrize("size,gain", [(4e-37, 1.0), (1e-35, 1.0), (1e-20, 1e-17), (1e-30, 1.0), (1e-33, 0.5)])
def test_rows_of_tiny_values_in_8_bits(bd, rows, cols, skip, off, size, gain):
    """y = h g / sqrt(mean h^2 + eps) is representable, down to 1e-34 here, and its 8 bits are those of larger rows."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    # (magnitudes of 0.5 to 2 times the size: the smallest, 2e-37, is a normal number, as FP32 arithmetic here flushes others)
    x = ((0.5 + 1.5 * torch.rand(rows, cols, device="cuda", generator=g)) * size).to(BF16)
    x *= torch.where(torch.rand(rows, cols, device="cuda", generator=g) < 0.5, -1, 1)
    x[:, 1] = 0
    w = torch.full((cols + 1,), gain, device="cuda", dtype=torch.float32)[1:]
    r = torch.zeros(rows, cols + 5, device="cuda", dtype=BF16)[:, 5:] if off else None
    got, scale, q = norm(bd, x, r, w, skip=skip)
    y = x.double() * w.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-6)
    assert ((scale.double() - y.abs().amax(1) / 448).abs() <= 1e-5 * y.abs().amax(1) / 448).all()
    # e4m3 rounding, 2^-4 of a value from 2^-6 on (all but the zeros are above 448 / 4)
    assert ((got - y).abs() <= (2.0 ** -4 + 2e-5) * y.abs()).all()
    assert (q[:, 1].float() == 0).all()


@pytest.mark.parametrize("rows,cols,skip", WIDTHS)
def test_rows_of_zeros_without_an_epsilon_have_scale_0(bd, rows, cols, skip):
    x = torch.ones(rows, cols, device="cuda", dtype=BF16)
    x[::2] = 0
    got, scale, q = norm(bd, x, eps=0.0, skip=skip)
    assert (scale[::2] == 0).all() and (q[::2].float() == 0).all()
    assert ((scale[1::2] * 448 - 1).abs() < 1e-5).all() and (q[1::2].float() == 448).all()


@pytest.mark.parametrize("cols", [2 ** 31 - 1, 2 ** 31 - 8192])
@pytest.mark.parametrize("out_dtype", ["BF16", "E4M3"])
def test_rows_whose_columns_pass_32_bits_are_refused(bd, cols, out_dtype):
    """(By the host, ahead of the addresses: nothing is launched.)"""
    p = bd.AddRmsNormParams(dtype=bd.BF16, rows=1, cols=cols, out_dtype=getattr(bd, out_dtype))
    assert bd.lib().bdattn_add_rmsnorm_fwd(p, None) == -1 and "columns" in bd.last_error()
    p.cols = 2 ** 31 - 8193
    assert bd.lib().bdattn_add_rmsnorm_fwd(p, None) == -1 and "null" in bd.last_error()
