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


def window_operands(segments):
    q, k = z(2, 3, 128), z(2, 9, 128)
    t = {"q": q, "k": k, "v": k.clone(), "out": q.clone(), "kv_len": z(2, dtype=torch.int32), "key_mask": z(9, dtype=torch.float32)}
    return t if not segments else {n: [x] if n in ("q", "k", "v", "out") else x for n, x in t.items()}


class OnGpu:
    """A tensor of the host that says it lies on a GPU."""

    def __init__(self, t, index):
        self._t, self._index = t, index

    def __getattr__(self, name):
        return getattr(self._t, name)

    def get_device(self):
        return self._index

    @property
    def is_cuda(self):
        return True


def test_segments_refuse_tensors_of_the_host(monkeypatch):
    monkeypatch.setattr(bd, "sdpa_fwd", lambda *a, **k: pytest.fail("an address of the host went to the library"))
    for host in ("q", "k", "v", "out", "kv_len", "key_mask", None):
        t = window_operands(True)
        if host is not None:               # all others on a GPU
            for name, x in t.items():
                if name != host:
                    t[name] = [OnGpu(x[0], 0)] if isinstance(x, list) else OnGpu(x, 0)
        with pytest.raises(bd.BdattnError, match="not on the GPU"):
            bd.sdpa_window_fwd(*(t[n] for n in ("q", "k", "v", "out")), 2, window=4, kv_len=t["kv_len"], key_mask=t["key_mask"])


def test_segments_refuse_tensors_of_different_gpus(monkeypatch):
    monkeypatch.setattr(bd, "sdpa_fwd", lambda *a, **k: pytest.fail("the library was asked"))
    for other in ("k", "v", "out", "kv_len", "key_mask"):
        t = {n: [OnGpu(x[0], int(n == other))] if isinstance(x, list) else OnGpu(x, int(n == other)) for n, x in window_operands(True).items()}
        with pytest.raises(bd.BdattnError, match="different GPUs"):
            bd.sdpa_window_fwd(*(t[n] for n in ("q", "k", "v", "out")), 2, window=4, kv_len=t["kv_len"], key_mask=t["key_mask"])


def test_tensors_of_another_gpu_than_the_current_one_are_refused():
    """What the calls ask about the GPUs of their tensors (the current one's number ahead of theirs; -1 is the host)."""
    one_gpu = (bd._binding or bd._load_binding()).one_gpu
    assert one_gpu(0, 0, 0, 0) is None and one_gpu(3, 3) is None
    for gpus, reason in (((0, 1, 1), "current GPU"), ((1, 0), "current GPU"), ((0, 0, 1), "different GPUs"), ((0, 0, -1), "not on the GPU"),
                         ((0, -1, 0), "not on the GPU")):
        with pytest.raises(bd.BdattnError, match=reason):
            one_gpu(*gpus)
    for bad in ((), ("0", 0), (0, None)):
        with pytest.raises(TypeError):
            one_gpu(*bad)


def test_segments_refuse_heads_that_do_not_divide_the_width():
    """264 columns are no 32 heads; the same call without segments refuses them too."""
    q, k = z(1, 3, 264), z(1, 9, 264)
    for args in (([q], [k], [k], [q]), (q, k, k, q)):
        for heads in (32, 5, 0, -1):
            with pytest.raises(bd.BdattnError, match="num_heads"):
                bd.sdpa_window_fwd(*args, heads, window=4)
