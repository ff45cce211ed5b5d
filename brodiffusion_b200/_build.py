"""Build recipe for ``libbdattn.so`` (nvcc, sm_100a only, in-tree output)."""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libbdattn.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "--use_fast_math",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]
UNITS = ["bdattn_lib", "bdattn_lib4"]      # translation units


# The Python module of the calls of a decoding step (csrc/binding.cpp): torch tensors in, the library's entry points out.
BINDING_PATH = os.path.join(PKG_DIR, "_binding.so")


def build_binding(force: bool = False):
    """Compile ``_binding.so``; without a torch that has CUDA there is nothing to bind (None), and the library stands alone."""
    src = os.path.join(CSRC, "binding.cpp")
    header = os.path.join(PKG_DIR, "..", "include", "bdattn.h")
    if not force and os.path.exists(BINDING_PATH) and os.path.getmtime(BINDING_PATH) >= max(map(os.path.getmtime, (src, header))):
        return BINDING_PATH
    import sysconfig
    try:
        import torch
    except ModuleNotFoundError as e:
        if e.name != "torch":
            raise
        return None
    if torch.version.cuda is None:
        return None
    from torch.utils import cpp_extension
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *[f"-I{p}" for p in cpp_extension.include_paths()], f"-I{cuda}/include", f"-I{sysconfig.get_paths()['include']}",
           src, "-o", BINDING_PATH, f"-L{PKG_DIR}", "-lbdattn", f"-L{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("building _binding.so failed")
    return BINDING_PATH


def sources():
    out = []
    for root, _, files in os.walk(CSRC):
        out += [os.path.join(root, f) for f in files if f.endswith((".cu", ".cuh", ".h"))]
    out.append(os.path.join(PKG_DIR, "..", "include", "bdattn.h"))
    return out


def is_stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(s) > t for s in sources())


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every CUDA source of the package into ``libbdattn.so``."""
    if not force and not is_stale():
        build_binding()
        return LIB_PATH
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    log, failed = "", False
    with tempfile.TemporaryDirectory() as d:
        # the units side by side, then one library of them
        objects = [os.path.join(d, u + ".o") for u in UNITS]
        cmds = [[nvcc, *NVCC_FLAGS, "-c", "-o", o, os.path.join(CSRC, u + ".cu")] for u, o in zip(UNITS, objects)]
        running = [subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for c in cmds]
        for cmd, p in zip(cmds, running):
            out = p.communicate()[0]
            log += " ".join(cmd) + "\n" + out
            failed = failed or p.returncode != 0
        if not failed:
            cmd = [nvcc, *NVCC_FLAGS, "-shared", "-o", LIB_PATH, *objects]
            res = subprocess.run(cmd, capture_output=True, text=True)
            log += " ".join(cmd) + "\n" + res.stdout + res.stderr
            failed = res.returncode != 0
    with open(os.path.join(PKG_DIR, "build.log"), "w") as f:
        f.write(log)
    if failed:
        sys.stderr.write(log)
        raise RuntimeError("nvcc failed building libbdattn.so")
    if verbose:
        print(log)
    build_binding(force)
    return LIB_PATH


if __name__ == "__main__":
    build(force=True, verbose=True)
