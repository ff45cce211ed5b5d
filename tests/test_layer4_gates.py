"""What a layer with weights and cache in 4 bits refuses ahead of its first call (no GPU)."""
import pytest
import torch

import brodiffusion_b200 as bd
from brodiffusion_b200 import layer as LY

BF16 = torch.bfloat16
D, NH, NKV, HD, F = 64, 2, 1, 64, 128


def z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def layer(monkeypatch, **more):
    monkeypatch.setattr(LY, "quantise_rows4", lambda w, group: None)
    f = torch.float32
    w = dict(norm1=z(D, dtype=f), norm2=z(D, dtype=f), post1=z(D, dtype=f), post2=z(D, dtype=f), wqkv=z((NH + 2 * NKV) * HD, D),
             wo=z(D, NH * HD), w_up=z(F, D), w_down=z(D, F), **more)
    return LY.FourBitLayer(w, NH, NKV, HD)


def nothing_is_called(monkeypatch):
    def call(*a, **kw):
        raise AssertionError("a call was made")
    for name in ("add_rmsnorm_fwd", "linear_w4_fwd", "rmsnorm_rope", "cache4_append", "cache4_read", "sdpa_cache4_fwd", "sdpa_window_fwd",
                 "sandwich_norm_fwd", "w4_unpack", "linear_act_fwd"):
        monkeypatch.setattr(bd, name, call)


@pytest.mark.parametrize("which", ["gate1", "gate2"])
@pytest.mark.parametrize("B,n,L", [(3, 2, 2), (3, 2, 1), (2, 4, 2), (2, 4, 4), (1, 3, 3)])
def test_gates_that_do_not_divide_the_sequences(monkeypatch, which, B, n, L):
    """n vectors are for B / n sequences each: rows alone would let a vector end inside a sequence."""
    layer4 = layer(monkeypatch, **{"gate1": z(D), "gate2": z(D), which: z(n, D)})
    nothing_is_called(monkeypatch)
    kv = LY.KvCache4(B, 16, NKV, HD, 32, BF16, device="cpu")
    with pytest.raises(bd.BdattnError, match="gate"):
        layer4.forward(z(B, L, D), kv, z(16, HD // 2), z(16, HD // 2))
    assert kv.filled == [0] * B and kv.lengths.tolist() == [0] * B


@pytest.mark.parametrize("odd", ["wqkv", "wo", "w_up", "w_down"])
def test_matrices_of_several_types(monkeypatch, odd):
    """Packed weights do not say of which type their pairs are."""
    monkeypatch.setattr(LY, "quantise_rows4", lambda w, group: None)
    w = dict(norm1=z(D), norm2=z(D), post1=z(D), post2=z(D), wqkv=z((NH + 2 * NKV) * HD, D), wo=z(D, NH * HD), w_up=z(F, D), w_down=z(D, F))
    LY.FourBitLayer(w, NH, NKV, HD)
    with pytest.raises(bd.BdattnError, match="dtype"):
        LY.FourBitLayer({**w, odd: w[odd].half()}, NH, NKV, HD)
    with pytest.raises(bd.BdattnError, match="dtype"):
        LY.FourBitLayer({**w, **{n: w[n].float() for n in ("wqkv", "wo", "w_up", "w_down")}}, NH, NKV, HD)


@pytest.mark.parametrize("L", [1, 40])
def test_a_stream_of_another_type_than_the_weights(monkeypatch, L):
    """(gains in FP32 fit both)"""
    layer4 = layer(monkeypatch)
    nothing_is_called(monkeypatch)
    kv = LY.KvCache4(2, 64, NKV, HD, 32, torch.float16, device="cpu")
    with pytest.raises(bd.BdattnError, match="dtype"):
        layer4.forward(z(2, L, D, dtype=torch.float16), kv, z(64, HD // 2), z(64, HD // 2))
    assert kv.filled == [0, 0] and kv.lengths.tolist() == [0, 0]


@pytest.mark.parametrize("D,F,rows,many", [(64, 128, 95, False), (64, 128, 96, True), (2048, 4096, 63, False), (2048, 4096, 64, True), (2040, 4096, 64, False)])
def test_matrices_that_go_back_to_16_bits(monkeypatch, D, F, rows, many):
    """Small ones half as many rows later."""
    monkeypatch.setattr(LY, "quantise_rows4", lambda w, group: None)
    w = dict(norm1=z(D), norm2=z(D), post1=z(D), post2=z(D), wqkv=z(3 * HD, D), wo=z(D, HD), w_up=z(F, D), w_down=z(D, F))
    made = []
    for name in ("linear_w4_fwd", "w4_unpack", "linear_act_fwd"):
        monkeypatch.setattr(bd, name, lambda *a, name=name, **kw: made.append(name))
    y = LY.FourBitLayer(w, 1, 1, HD)._product(z(rows, D), "w_up")
    assert y.shape == (rows, F) and made == (["w4_unpack", "linear_act_fwd"] if many else ["linear_w4_fwd"])
