"""Operands of a layer's operators that the library cannot take as they are: refused by the binding, with the reason,
before the library sees an address (no GPU)."""
import pytest
import torch

import brodiffusion_b200 as bd

BF16 = torch.bfloat16


def z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


# An expanded row has a stride of zero, which stands for dense rows in the library's structures: it would be read, or
# written, past its end.  The message is compared, since tensors of the host are refused after these.
@pytest.mark.parametrize("operand", ["x", "residual", "residual_out", "out"])
def test_norm_refuses_rows_that_are_the_same_memory(operand):
    t = {name: z(4, 64) for name in ("x", "residual", "residual_out", "out")}
    t[operand] = z(1, 64).expand(4, 64)
    with pytest.raises(bd.BdattnError, match=f"^{operand} .*rows overlap"):
        bd.add_rmsnorm_fwd(t["x"], t["out"], residual=t["residual"], residual_out=t["residual_out"])


@pytest.mark.parametrize("operand", ["x", "w", "residual", "y"])
def test_linear_refuses_rows_that_are_the_same_memory(operand):
    shapes = {"x": (4, 64), "w": (32, 64), "residual": (4, 32), "y": (4, 32)}
    t = {name: z(*s) for name, s in shapes.items()}
    t[operand] = z(1, shapes[operand][1]).expand(shapes[operand])
    with pytest.raises(bd.BdattnError, match=f"^{operand} .*rows overlap"):
        bd.linear_act_fwd(t["x"], t["w"], None, t["y"], residual=t["residual"])


def test_rows_that_overlap_in_part_and_a_single_row_of_any_stride():
    with pytest.raises(bd.BdattnError, match="^x .*rows overlap"):
        bd.add_rmsnorm_fwd(z(256).as_strided((4, 64), (32, 1)), z(4, 64))
    with pytest.raises(bd.BdattnError, match="GPU"):             # nothing else to refuse: a row is dense whatever its stride
        bd.add_rmsnorm_fwd(z(64).as_strided((1, 64), (0, 1)), z(1, 64))
