"""Builds ``lib/libflashsinkhorn_b200.so`` from ``csrc/*.cu`` with nvcc for sm_100a (in-tree), and beside it the torch
binding of the routed-experts operators, ``lib/fs_torch.so``, from ``csrc/fs_torch.cpp`` with the host compiler.

    python -m flash_sinkhorn_b200.build_ext [--force] [--verbose]

nvcc cross-compiles without a GPU. The library links the CUDA runtime statically and
resolves the one driver entry point it needs (tensor-map encoding) at run time, so it
has no load-time dependency beyond libstdc++. The binding is compiled against the torch that is installed.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "lib", "libflashsinkhorn_b200.so")
BINDING = os.path.join(HERE, "lib", "fs_torch.so")
BINDING_SOURCE = "fs_torch.cpp"
SOURCES = ["fs_api.cu", "fs_simt.cu", "fs_tc.cu", "fs_tck.cu", "fs_sym.cu", "fs_static.cu", "fs_micro.cu",
           "fs_experts.cu", "fs_group.cu", "fs_norm.cu", "fs_mm8.cu", "fs_ortho.cu", "fs_health.cu"]
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
]


def _stale(out: str, sources) -> bool:
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    deps = list(sources) + [os.path.join(os.path.dirname(HERE), "include", "flash_sinkhorn_b200.h"), os.path.abspath(__file__)]
    return any(os.path.getmtime(p) > t for p in deps if os.path.isfile(p))


def _run(cmd, out: str, verbose: bool) -> None:
    """Runs a compiler into a file of this process's own, which then takes the place of ``out``."""
    part = f"{out}.{os.getpid()}.o"
    res = subprocess.run(cmd + ["-o", part], capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode}): {' '.join(cmd)}")
    os.replace(part, out)


def build_binding(force: bool = False, verbose: bool = False) -> str:
    source = os.path.join(CSRC, BINDING_SOURCE)
    if not force and not _stale(BINDING, [source]):
        return BINDING
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(shutil.which(os.environ.get("NVCC", "nvcc")) or "/usr/local/cuda/bin/nvcc"))), "include")
    # the compiler that nvcc takes, whatever $CXX says: one that links its C++ run-time library statically brings a second
    # copy into the process, whose streams crash
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for path in cpp_extension.include_paths() + [cuda, sysconfig.get_paths()["include"]]:
        cmd += ["-isystem", path]
    cmd += [source, f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    os.makedirs(os.path.dirname(BINDING), exist_ok=True)
    _run(cmd, BINDING, verbose)
    return BINDING


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the sources side by side and links them; the binding at the same time."""
    from concurrent.futures import ThreadPoolExecutor

    sources = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f != BINDING_SOURCE]
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    with ThreadPoolExecutor(os.cpu_count() or 4) as pool:
        binding = pool.submit(build_binding, force, verbose)
        if force or _stale(OUT, sources):
            nvcc = [os.environ.get("NVCC", "nvcc")] + FLAGS
            with tempfile.TemporaryDirectory() as folder:
                objects = [os.path.join(folder, s[:-3] + ".o") for s in SOURCES]
                options = ["-Xptxas", "-v"] if verbose else []
                list(pool.map(lambda s, o: _run(nvcc + options + ["-c", os.path.join(CSRC, s)], o, verbose), SOURCES, objects))
                _run(nvcc + ["-shared"] + objects, OUT, verbose)
        binding.result()
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
