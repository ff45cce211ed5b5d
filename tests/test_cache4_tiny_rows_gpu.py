"""Rows of tiny BF16 values into the 4-bit cache: steps and codes are the format's to the bit, as for values of any other size."""
import pytest
import torch

from four_bit import by_heads, flat, held, quantised, randn
from test_cache4_gpu import SHAPES, garbage, read

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,group", SHAPES)
@pytest.mark.parametrize("exponent", [-60, -70, -90, -101, -104, -110, -118])
def test_rows_of_tiny_values(bd, exponent, hd, group):
    """Among some hundred rows there are quotients on the border between two codes, and fifteenths on that of two steps."""
    heads, rows = 2, 700
    x = (randn(1, 1, rows, heads * hd, dtype=torch.float32) * 2.0 ** exponent).bfloat16()
    x[0, ::2] = (torch.randint(-40, 40, (rows // 2, heads * hd), device="cuda", generator=torch.Generator("cuda").manual_seed(2)) * 2.0 ** (exponent - 3)).bfloat16()
    c = garbage(bd, 1, heads, rows, hd, group, torch.bfloat16)
    bd.cache4_append(x, x, c)
    want = quantised(by_heads(x, heads), group)[1]
    assert (want[..., 0] >= 2.0 ** -126).all()
    for scales in (c.k_scales, c.v_scales):
        assert (scales == want).all()
    for got in read(bd, c, rows):
        assert (got == flat(held(by_heads(x, heads), group)).to(x.dtype)).all()


def test_groups_beside_one_another(bd):
    """Tiny groups between ordinary ones and large ones, rows alike but for a power of two: the same codes."""
    hd, group, rows = 128, 32, 200
    x = randn(3, 1, rows, hd, dtype=torch.float32)
    x = (x * 2.0 ** torch.tensor([-110.0, 0.0, 100.0, -64.0], device="cuda").repeat_interleave(group)).bfloat16()
    c = garbage(bd, 1, 1, rows, hd, group, torch.bfloat16)
    bd.cache4_append(x, x, c)
    for got in read(bd, c, rows):
        assert (got == flat(held(by_heads(x, 1), group)).to(x.dtype)).all()
