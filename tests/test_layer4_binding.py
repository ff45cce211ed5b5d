"""The structures of the 4-bit operators against the header, what the binding refuses before the library is asked, a layer's
cache when one of its calls is refused, and loads past the read-only path (no GPU)."""
import ctypes as C
import os
import re
import subprocess
import tempfile

import pytest
import torch

import brodiffusion_b200 as bd
from brodiffusion_b200 import layer as LY

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTURES = [(bd.SandwichNormParams, "bdattn_sandwich_norm_params"), (bd.LinearW4Params, "bdattn_linear_w4_params"),
              (bd.Cache4Params, "bdattn_cache4"), (bd.Cache4Rows, "bdattn_cache4_rows"), (bd.SdpaCache4Params, "bdattn_sdpa_cache4_params")]
BF16 = torch.bfloat16


def test_mirrors_match_the_header():
    lines = ['printf("%s %%zu\\n", sizeof(%s));' % (name, name) for _, name in STRUCTURES]
    lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, f, name, f) for cls, name in STRUCTURES for f, _ in cls._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"bdattn.h\"\nint main(void) { " + " ".join(lines) + " return 0; }\n"
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "s.c"), "w") as f:
            f.write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "s.c"), "-o", os.path.join(d, "s")])
        said = dict(line.split() for line in subprocess.check_output([os.path.join(d, "s")], text=True).splitlines())
    for cls, name in STRUCTURES:
        assert int(said[name]) == C.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(said[f"{name}.{f}"]) == getattr(cls, f).offset


def test_bytes_of_packed_weights():
    assert bd.w4_bytes(16, 128, 32) == 1024 + 256 and bd.w4_bytes(17, 129, 128) == 4 * (1024 + 64) and bd.w4_bytes(1, 8, 64) == 1024 + 128
    for bad in ((0, 8, 32), (8, 0, 32), (-1, 8, 32), (8, 8, 0), (8, 8, 256)):
        assert bd.w4_bytes(*bad) == 0
    assert bd.w4_bytes(1 << 20, 1 << 20, 32) == (1 << 16) * (1 << 13) * 1280


def z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def cache(b=2, h=2, rows=16, hd=64, group=32, dtype=BF16):
    return bd.Cache4.empty(b, h, rows, hd, group, dtype, device="cpu")


def changed(c, **kw):
    return bd.Cache4(*(kw.get(n, getattr(c, n)) for n in bd.Cache4.__slots__))


def test_shapes_that_do_not_fit_are_refused_before_any_launch():
    x, y, c = z(4, 64), z(4, 32), cache()
    w = z(bd.w4_bytes(32, 64, 32), dtype=torch.uint8)
    q, k = z(2, 3, 256), z(2, 3, 128)
    wide = cache(4, 4, 16)
    for call in (lambda: bd.sandwich_norm_fwd(x, x[:2], x), lambda: bd.sandwich_norm_fwd(x, x, x[:, :32]),
                 lambda: bd.sandwich_norm_fwd(x, x, x, out=x[:, :32]), lambda: bd.sandwich_norm_fwd(x, x, x, x[0, :8]),
                 lambda: bd.sandwich_norm_fwd(x, x.float(), x), lambda: bd.sandwich_norm_fwd(x, x, x, gate=z(2, 32)),
                 lambda: bd.sandwich_norm_fwd(x, x, x, gate=z(0, 64)), lambda: bd.sandwich_norm_fwd(x, z(1, 64).expand(4, 64), x),
                 lambda: bd.sandwich_norm_fwd(x, x, x, gate=z(1, 64).expand(2, 64)),
                 lambda: bd.sandwich_norm_fwd(x, x, x, z(64), gain=z(64).float(), out=x),
                 lambda: bd.linear_w4_fwd(x, w, None, y, group=64), lambda: bd.linear_w4_fwd(x, w[:-1], None, y, group=32),
                 lambda: bd.linear_w4_fwd(x, w.float(), None, y, group=32), lambda: bd.linear_w4_fwd(x[:2], w, None, y, group=32),
                 lambda: bd.linear_w4_fwd(x, w, None, y, group=32, act="tanh"), lambda: bd.linear_w4_fwd(x, w, y[0, :8], y, group=32),
                 lambda: bd.linear_w4_fwd(z(1, 64).expand(4, 64), w, None, y, group=32), lambda: bd.linear_w4_fwd(x, w, None, y, group=32, residual=y.half()),
                 lambda: bd.w4_pack(z(32, 32, dtype=torch.uint8), z(32, 3, 2), w, group=32),
                 lambda: bd.w4_pack(z(32, 32, dtype=torch.uint8), z(32, 2, 2).float(), w, group=32),
                 lambda: bd.w4_pack(z(32, 32, dtype=torch.uint8), z(32, 2, 2), w[1:], group=32),
                 lambda: bd.w4_pack(z(32, 32, dtype=torch.uint8), z(1, 2, 2).expand(32, 2, 2), w, group=32),
                 lambda: bd.w4_unpack(w[1:], z(32, 64), group=32), lambda: bd.w4_unpack(w, z(32, 64), group=64),
                 lambda: bd.w4_unpack(w, z(32, 136), group=32), lambda: bd.w4_unpack(w, z(32, 64).int(), group=32),
                 lambda: bd.w4_unpack(w, z(1, 64).expand(32, 64), group=32),
                 lambda: bd.cache4_append(k, k[:, :2], c), lambda: bd.cache4_append(k[:1], k[:1], c), lambda: bd.cache4_append(q, q, c),
                 lambda: bd.cache4_append(k.half(), k.half(), c), lambda: bd.cache4_append(k, k, c, kv_len=z(2)),
                 lambda: bd.cache4_append(k, k, c, kv_len=z(3, dtype=torch.int32)),
                 lambda: bd.cache4_append(k, k[:1].expand(2, 3, 128), c),
                 lambda: bd.cache4_append(k, k, changed(c, v_codes=c.v_codes[:, :, :8])),
                 lambda: bd.cache4_append(k, k, changed(c, k_scales=c.k_scales[:, :, :8], v_scales=c.v_scales[:, :, :8])),
                 lambda: bd.cache4_append(k, k, changed(c, v_codes=wide.v_codes[::2, ::2])),                # other strides than K
                 lambda: bd.cache4_append(k, k, bd.Cache4(*(getattr(c, n).transpose(1, 2) for n in bd.Cache4.__slots__))),
                 lambda: bd.sdpa_cache4_fwd(q, c, q[:, :2], 4), lambda: bd.sdpa_cache4_fwd(q, c, q, 2), lambda: bd.sdpa_cache4_fwd(q, c, q, 0),
                 lambda: bd.sdpa_cache4_fwd(q[:1], c, q[:1], 4), lambda: bd.sdpa_cache4_fwd(q, c, q, 4, key_mask=z(15).float())):
        with pytest.raises(bd.BdattnError) as e:
            call()
        assert "not on the GPU" not in str(e.value)
    for call in (lambda: bd.sandwich_norm_fwd(None, x, x), lambda: bd.sandwich_norm_fwd(x, x, x, eps="a"), lambda: bd.linear_w4_fwd(x, w, None, y, group="32"),
                 lambda: bd.sdpa_cache4_fwd(q, c, q, 4, window=2.0), lambda: bd.sdpa_cache4_fwd(q, c, q, 4, window=1 << 40),
                 lambda: bd.cache4_append(k, [1], c)):
        with pytest.raises(TypeError):
            call()
    # tensors of the host are refused before the library sees their addresses
    for call in (lambda: bd.sandwich_norm_fwd(x, x, x), lambda: bd.linear_w4_fwd(x, w, None, y, group=32), lambda: bd.cache4_append(k, k, c),
                 lambda: bd.cache4_read(c, k, k), lambda: bd.sdpa_cache4_fwd(q, c, q, 4),
                 lambda: bd.w4_pack(z(32, 32, dtype=torch.uint8), z(32, 2, 2), w, group=32), lambda: bd.w4_unpack(w, z(32, 64), group=32)):
        with pytest.raises(bd.BdattnError, match="GPU"):
            call()


def test_a_view_of_the_first_rows():
    c = cache()
    f = c.first(5)
    assert c.rows == 16 and f.rows == 5 and f.k_codes.data_ptr() == c.k_codes.data_ptr() and f.v_scales.shape == (2, 2, 5, 2, 2)


CALLS = ["add_rmsnorm_fwd", "linear_w4_fwd", "rmsnorm_rope", "cache4_append", "cache4_read", "sdpa_cache4_fwd", "sdpa_window_fwd", "sandwich_norm_fwd",
         "w4_unpack", "linear_act_fwd"]


@pytest.mark.parametrize("new", [2, 40])
@pytest.mark.parametrize("refused", range(16))
def test_a_refused_call_leaves_the_cache_as_it_was(monkeypatch, refused, new):
    D, nh, nkv, hd, F, B = 64, 2, 1, 64, 128, 3
    monkeypatch.setattr(LY, "quantise_rows4", lambda w, group: None)
    w = dict(norm1=z(D), norm2=z(D), post1=z(D), post2=z(D), wqkv=z((nh + 2 * nkv) * hd, D), wo=z(D, nh * hd), w_up=z(F, D), w_down=z(D, F))
    L = LY.FourBitLayer(w, nh, nkv, hd, window=4)
    kv = LY.KvCache4(B, 64, nkv, hd, 32, BF16, device="cpu")
    kv.filled, lengths = [5, 0, 9], kv.lengths
    lengths.copy_(torch.tensor(kv.filled))
    made = []

    def stand_in(name):
        def call(*args, **kw):
            made.append(name)
            if "kv_len" in kw:
                assert kw["kv_len"].tolist() == [5 + new, new, 9 + new]           # the new rows are seen
            if len(made) == refused + 1:
                raise bd.BdattnError("refused")
        return call
    for name in CALLS:
        monkeypatch.setattr(bd, name, stand_in(name))
    cos = torch.zeros(64, hd // 2)
    x = z(B, new, D)
    assert 2 < L.PROMPT <= 40 and 2 * B < L.MANY <= 40 * B
    calls = 11 if new == 2 else 16
    if refused < calls:
        with pytest.raises(bd.BdattnError, match="refused"):
            L.forward(x, kv, cos, cos)
        assert kv.filled == [5, 0, 9] and kv.lengths is lengths and lengths.tolist() == [5, 0, 9]
    made[:] = ["no more"] * 20
    L.forward(x, kv, cos, cos)
    assert kv.filled == [5 + new, new, 9 + new] and lengths.tolist() == kv.filled
    product = ["linear_w4_fwd"] if new == 2 else ["w4_unpack", "linear_act_fwd"]
    assert made[20:] == ["add_rmsnorm_fwd", *product, "rmsnorm_rope", "rmsnorm_rope", "cache4_append"] + \
        (["sdpa_cache4_fwd"] if new == 2 else ["cache4_read", "sdpa_window_fwd"]) + \
        [*product, "sandwich_norm_fwd", *product, *product, "sandwich_norm_fwd"]


# These kernels run before the kernel ahead of them has ended, and may not read what it writes through the read-only path.
@pytest.mark.parametrize("name", ["norm_rows.cuh", "sandwich_norm.cu", "four_bit.cuh", "w4_linear.cu", "cache4.cu", "sdpa_cache4.cu"])
def test_operands_are_not_read_through_the_read_only_path(name):
    with open(os.path.join(ROOT, "brodiffusion_b200", "csrc", name)) as f:
        code = [line.split("//")[0] for line in f]
    assert [line for line in code if re.search(r"__ldg\s*\(|ld\.global\.nc|__restrict__", line)] == []
