"""Builds libdflash_b200.so in-tree with nvcc for sm_100a (the only supported target)."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG = CSRC.parent
LIB = PKG / "libdflash_b200.so"
BINDING = PKG / "_native.so"
BINDING_STAMP = CSRC / "build" / "_native.torch"   # the torch that BINDING was built against
SOURCES = ["runtime.cu", "qmm.cu", "qmm_tc.cu", "gdn.cu", "gdn_layer.cu", "sdpa.cu", "sdpa_tc.cu", "glue.cu", "peer.cu", "kv4.cu",
           "kv4_tc.cu", "logprobs.cu"]
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "--use_fast_math",
         "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "-Xptxas", "-v"]
# Sources whose results are defined to the last bit, subnormals included: IEEE division and no flush to zero.
IEEE_SOURCES = {"kv4.cu", "kv4_tc.cu"}


def _nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found: the dflash B200 library cannot be built")
    return nvcc


def _stale(obj: Path, src: Path) -> bool:
    if not obj.exists():
        return True
    newest = max(p.stat().st_mtime for p in [src, *CSRC.glob("*.cuh"), PKG.parent / "include" / "dflash_b200.h"])
    return obj.stat().st_mtime < newest


def _into_place(target: Path, run) -> subprocess.CompletedProcess:
    """``run(path)`` writes a file that replaces ``target`` in one step where it succeeds: another process finds the old file or the
    new one, never a part."""
    part = target.with_name(f".{target.name}.{os.getpid()}")
    try:
        res = run(str(part))
        if res.returncode == 0:
            os.replace(part, target)
        return res
    finally:
        part.unlink(missing_ok=True)


def binding_fits() -> bool:
    """Whether the binding is there and was not built against another torch than the installed one."""
    import torch
    return BINDING.exists() and (not BINDING_STAMP.exists() or BINDING_STAMP.read_text() == str(torch.__version__))


def build_binding(force: bool = False) -> Path:
    """The C++ binding of the operators in quantized_kv.py and logprobs.py, against the installed torch."""
    src = CSRC / "binding.cpp"
    if not force and binding_fits() and not _stale(BINDING, src):
        return BINDING
    import torch
    base = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    res = _into_place(BINDING, lambda out: subprocess.run(
        ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
         f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{base}/include",
         f"-I{base}/include/torch/csrc/api/include", f"-I{cuda}/include", f"-I{sysconfig.get_paths()['include']}", str(src), "-o",
         out, f"-L{base}/lib", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"], capture_output=True, text=True))
    if res.returncode != 0:
        sys.stderr.write(res.stderr)
        raise RuntimeError("g++ failed on binding.cpp")
    BINDING_STAMP.parent.mkdir(exist_ok=True)
    BINDING_STAMP.write_text(str(torch.__version__))
    return BINDING


def build(force: bool = False, verbose: bool = False) -> Path:
    nvcc = _nvcc()
    objdir = CSRC / "build"
    objdir.mkdir(exist_ok=True)
    objs, rebuilt = [], False
    for name in SOURCES:
        src = CSRC / name
        if not src.exists():
            continue
        obj = objdir / (src.stem + ".o")
        if force or _stale(obj, src):
            flags = [f for f in FLAGS if f != "--use_fast_math" or name not in IEEE_SOURCES]
            cmd = [nvcc, *flags, "-c", str(src), "-o", str(obj)]
            res = subprocess.run(cmd, capture_output=True, text=True)
            (objdir / (src.stem + ".ptxas.txt")).write_text(res.stderr)
            if res.returncode != 0:
                sys.stderr.write(res.stderr)
                raise RuntimeError(f"nvcc failed on {name}")
            if verbose:
                sys.stderr.write(res.stderr)
            rebuilt = True
        objs.append(str(obj))
    if rebuilt or not LIB.exists():
        res = _into_place(LIB, lambda out: subprocess.run([nvcc, "-shared", "-o", out, *objs, "-lcudart", "-Xlinker", "--no-undefined"],
                                                          capture_output=True, text=True))
        if res.returncode != 0:
            sys.stderr.write(res.stderr)
            raise RuntimeError("link of libdflash_b200.so failed")
    build_binding(force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
