"""Build libpkb200.so in-tree for sm_100a (nvcc cross-compiles without a GPU)."""
from __future__ import annotations

import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "_lib", "libpkb200.so")
SOURCES = ["pkb200", "paged"]


def build_binding(verbose: bool = False) -> str:
    """The Python module of the paged-cache operators (host code only), next to the library."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    out = os.path.join(os.path.dirname(OUT), "_paged" + sysconfig.get_config_var("EXT_SUFFIX"))
    cuda = os.path.join(os.path.dirname(os.path.dirname(shutil.which("nvcc"))), "include")
    includes = cpp_extension.include_paths() + [cuda, sysconfig.get_paths()["include"]]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(arg for path in includes for arg in ("-isystem", path)), "-o", out,
           os.path.join(CSRC, "paged_binding.cpp"), "-L" + os.path.dirname(OUT), "-lpkb200", "-L" + libs,
           "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True, cwd=CSRC)
    return out


def build(verbose: bool = False) -> str:
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    arch = ["nvcc", "-gencode", "arch=compute_100a,code=sm_100a"]
    flags = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC"]
    objects = [os.path.join(os.path.dirname(OUT), name + ".o") for name in SOURCES]
    steps = [arch + flags + ["-c", "-o", obj, os.path.join(CSRC, name + ".cu")]
             for name, obj in zip(SOURCES, objects)]
    link = arch + ["-Xcompiler", "-fPIC", "-shared", "-o", OUT, *objects, "-lcudart"]
    if verbose:
        print("\n".join(" ".join(cmd) for cmd in steps + [link]))
    running = [subprocess.Popen(cmd, cwd=CSRC) for cmd in steps]  # side by side
    if any([p.wait() for p in running]):
        raise RuntimeError("pkb200: nvcc failed")
    subprocess.run(link, check=True, cwd=CSRC)
    build_binding(verbose)
    # the .npy launcher harness (reference cuda_run command line) over the library
    harness = ["nvcc", "-Wno-deprecated-gpu-targets", "-O2", "-std=c++17", "-o", os.path.join(os.path.dirname(OUT), "cuda_run"),
               os.path.join(CSRC, "cuda_run.cpp"), "-L" + os.path.dirname(OUT), "-lpkb200",
               "-lcudart", "-Xlinker", "-rpath=$ORIGIN"]
    if verbose:
        print(" ".join(harness))
    subprocess.run(harness, check=True, cwd=CSRC)
    return OUT


if __name__ == "__main__":
    print(build(verbose=True))
