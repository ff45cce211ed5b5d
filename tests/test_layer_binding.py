"""The packed parameter structures of a layer's operators against their ctypes mirrors, the mirrors against the header,
and what the binding refuses before the library is asked (no GPU)."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

import brodiffusion_b200 as bd

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTURES = [(bd.AddRmsNormParams, "bdattn_add_rmsnorm_params"), (bd.WindowParams, "bdattn_window_params"),
              (bd.LinearActParams, "bdattn_linear_act_params")]


def test_packed_window_is_the_structure():
    got = bd.WindowParams.from_buffer_copy(bd._pack_window(3, 1001, 1 << 40))
    assert (got.window, got.sinks, got.kv_len) == (3, 1001, 1 << 40)


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


def test_c_functions_take_their_own_structures_only():
    L = bd.lib()
    calls = {"bdattn_add_rmsnorm_fwd": (bd.AddRmsNormParams, lambda f, p: f(p, None)),
             "bdattn_linear_act_fwd": (bd.LinearActParams, lambda f, p: f(p, None)),
             "bdattn_sdpa_window_fwd": (bd.WindowParams, lambda f, p: f(bd.SdpaParams(), p, None))}
    for name, (cls, call) in calls.items():
        fn, own = getattr(L, name), cls()
        for p in (None, own, C.byref(own), C.pointer(own)):
            assert call(fn, p) == -1            # null or all zeros: refused by the entry point itself
        for p in (bd.QkvoParams(), bytes(own), 4096, "x"):
            with pytest.raises(C.ArgumentError):
                call(fn, p)


def test_shapes_that_do_not_fit_are_refused_before_any_launch():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16)
    y, w2 = torch.zeros(4, 32, dtype=torch.bfloat16), w
    for call in (lambda: bd.add_rmsnorm_fwd(x, x[:, :32]), lambda: bd.add_rmsnorm_fwd(x, x, w[0, :32]),
                 lambda: bd.add_rmsnorm_fwd(x, x, residual=w), lambda: bd.add_rmsnorm_fwd(x[0], x[0]),
                 lambda: bd.add_rmsnorm_fwd(x, x.to(torch.float8_e4m3fn), out_scale=torch.zeros(4, dtype=torch.float64)),
                 lambda: bd.linear_act_fwd(x, w, None, x), lambda: bd.linear_act_fwd(x, w[:, :32], None, y),
                 lambda: bd.linear_act_fwd(x, w, y[0, :8], y), lambda: bd.linear_act_fwd(x, w, None, y, act="tanh"),
                 lambda: bd.linear_act_fwd(x, w, None, y, x_scale=torch.zeros(5)),
                 lambda: bd.linear_act_fwd(x, w, None, y, residual=y.half())):
        with pytest.raises(bd.BdattnError):
            call()
    q, k = torch.zeros(2, 3, 128, dtype=torch.bfloat16), torch.zeros(2, 9, 64, dtype=torch.bfloat16)
    good = dict(window=4, num_kv_heads=1)
    for call in (lambda: bd.sdpa_window_fwd(q, k[:, :, :32], k[:, :, :32], q, 2, **good),      # heads of another width
                 lambda: bd.sdpa_window_fwd(q, k, k[:, :5], q, 2, **good),
                 lambda: bd.sdpa_window_fwd(q, k, k, q[:, :, :64], 2, **good),
                 lambda: bd.sdpa_window_fwd(q, k, k, q, 2, window=4),
                 lambda: bd.sdpa_window_fwd(q, k[:1], k[:1], q, 2, **good),
                 lambda: bd.sdpa_window_fwd(q, [k, k[:, :, :32]], [k, k], q, 2, **good),
                 lambda: bd.sdpa_window_fwd(q, k, k, q, 2, kv_len=torch.zeros(2), **good),
                 lambda: bd.sdpa_window_fwd(q, k, k, q, 2, kv_len=torch.zeros(3, dtype=torch.int32), **good),
                 lambda: bd.sdpa_window_fwd(q, k, k, q, 2, key_mask=torch.zeros(8), **good),
                 lambda: bd.sdpa_window_fwd(q, k[:1].expand(2, 9, 64), k, q, 2, **good),         # one sequence's rows for two
                 lambda: bd.sdpa_window_fwd([q], [k[:1].expand(2, 9, 64)], [k], [q], 2, **good)):
        with pytest.raises(bd.BdattnError):
            call()
    for w in (2.0, "4", None, 1 << 40):
        with pytest.raises(TypeError):
            bd.sdpa_window_fwd(q, k, k, q, 2, window=w, num_kv_heads=1)
        with pytest.raises(TypeError):
            bd.sdpa_window_fwd([q], [k], [k], [q], 2, window=w, num_kv_heads=1)
    for call in (lambda: bd.add_rmsnorm_fwd(None, x), lambda: bd.add_rmsnorm_fwd(x, x, 1.0), lambda: bd.add_rmsnorm_fwd(x, x, eps="a"),
                 lambda: bd.linear_act_fwd(x, [1], None, y), lambda: bd.sdpa_window_fwd(q, k, k, q, 2, kv_len=[1, 2], **good)):
        with pytest.raises(TypeError):
            call()
    # tensors of the host are refused before the library sees their addresses
    for call in (lambda: bd.add_rmsnorm_fwd(x, x), lambda: bd.linear_act_fwd(x, w2, None, y), lambda: bd.sdpa_window_fwd(q, k, k, q, 2, **good)):
        with pytest.raises(bd.BdattnError, match="GPU"):
            call()


def test_missing_module_is_reported(monkeypatch, tmp_path):
    monkeypatch.setattr(bd, "_binding", None)
    monkeypatch.setattr(bd._build, "BINDING_PATH", str(tmp_path / "nope.so"))
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    with pytest.raises(bd.BdattnError, match="missing"):
        bd.add_rmsnorm_fwd(x, x)
