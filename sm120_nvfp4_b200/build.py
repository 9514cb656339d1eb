"""Compile the CUDA sources of this package for sm_100a into one shared library.

    python -m sm120_nvfp4_b200.build            # builds sm120_nvfp4_b200/libb200_nvfp4.so

The library is built in-tree (it is git-ignored) and exports the C ABI declared in
include/b200_nvfp4.h plus the C++ API of include/sm120_nvfp4/. nvcc cross-compiles without a
GPU. cudart is linked statically; nothing else is linked (the driver entry point used to
encode tensor maps is fetched at run time).
"""
from __future__ import annotations

import hashlib
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OUT = PKG / "libb200_nvfp4.so"
SOURCES = ["gemm.cu", "gemm_splitk_static.cu", "gemm_host.cu", "fp8_gemm.cu", "fp8_quant.cu", "router_loss.cu", "router_grad.cu", "moe_kernels.cu", "ep_kernels.cu", "fused_moe.cu", "host_common.cpp", "api.cpp"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC,-fvisibility=hidden", "-Xptxas", "-v",
              f"-I{ROOT / 'include'}", f"-I{CSRC}"]


CALLS = PKG / ("_calls" + sysconfig.get_config_var("EXT_SUFFIX"))
CALLS_MADE_FROM = PKG / "build" / "_calls.digest"
_CALLS_SOURCE = CSRC / "torch_calls.cpp"
_CALLS_FLAGS = ["-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden"]


def _nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(cuda_home) / "bin" / "nvcc"
    return str(cand) if cand.exists() else "nvcc"


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> Path:
    headers = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.hpp")) + list((ROOT / "include").rglob("*.h*"))
    objdir = PKG / "build"
    objdir.mkdir(exist_ok=True)
    jobs = []
    for name in SOURCES:
        src = CSRC / name
        obj = objdir / (name + ".o")
        if force or _stale(obj, [src, *headers]):
            jobs.append((src, obj))

    def compile_one(job):
        src, obj = job
        flags = list(NVCC_FLAGS)
        if src.name == "api.cpp":  # the C++ API symbols are part of the public surface
            flags[flags.index("-fPIC,-fvisibility=hidden")] = "-fPIC"
        cmd = [_nvcc(), *flags, "-x", "cu", "-c", str(src), "-o", str(obj)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
        return src.name, res.stderr

    with ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
        for name, log in pool.map(compile_one, jobs):
            (objdir / (name + ".ptxas.log")).write_text(log)
            if verbose:
                print(f"== {name}\n{log}")
    objs = [objdir / (n + ".o") for n in SOURCES]
    if force or jobs or _stale(OUT, objs):
        cmd = [_nvcc(), "-shared", "-o", str(OUT), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    return OUT


def _calls_digest() -> str:
    """Of everything the extension module is made from: its source, the C ABI, torch, the interpreter, the flags."""
    import torch
    h = hashlib.sha256()
    for part in (_CALLS_SOURCE.read_bytes(), (ROOT / "include" / "b200_nvfp4.h").read_bytes(), torch.__version__.encode(),
                 sys.version.encode(), " ".join(_CALLS_FLAGS).encode()):
        h.update(hashlib.sha256(part).digest())
    return h.hexdigest()


def build_calls(force: bool = False) -> Path:
    """The extension module of csrc/torch_calls.cpp: host code only, against the installed torch and this
    package's library (found beside it at run time). Built again where what it was made from has changed; several
    processes may do so at once."""
    made_from = CALLS_MADE_FROM.read_text() if CALLS_MADE_FROM.exists() else ""
    digest = _calls_digest()
    if CALLS.exists() and made_from == digest and not force:
        return CALLS
    import torch
    from torch.utils import cpp_extension
    lib = OUT if OUT.exists() else build()
    includes = [*cpp_extension.include_paths(), os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include"),
                sysconfig.get_path("include"), str(ROOT / "include")]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    made = CALLS.with_name(f"{CALLS.name}.{os.getpid()}")
    cmd = ["g++", *_CALLS_FLAGS, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{i}" for i in includes),
           str(_CALLS_SOURCE), "-o", str(made), f"-L{libs}", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-lc10_cuda",
           "-lc10", f"-L{lib.parent}", f"-l:{lib.name}", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{libs}"]
    try:
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"g++ failed for {_CALLS_SOURCE.name}:\n{res.stdout}\n{res.stderr}")
        os.replace(made, CALLS)              # whole or not at all, for a process that loads it meanwhile
    finally:
        made.unlink(missing_ok=True)
    CALLS_MADE_FROM.parent.mkdir(exist_ok=True)
    CALLS_MADE_FROM.write_text(digest)
    return CALLS


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_calls(force="--force" in sys.argv))
