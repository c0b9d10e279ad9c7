"""Build recipe for the in-tree CUDA libraries (sm_100a only).

    python -m fav4_bshd.build [--force]

Compiles csrc/fav4_bshd.cu and csrc/paged.cu -> build/libfav4_bshd.so (the C
ABI of include/fav4_bshd.h) and csrc/probe.cu -> build/libfav4_probe.so (test probes)
with nvcc for sm_100a, statically linked against the CUDA runtime. The ptxas
resource report (registers, spills, shared memory) of each build is written
next to the library as build/<lib>.ptxas.txt. csrc/paged_torch.cpp ->
build/fav4_paged_torch.so is the PyTorch binding of the paged cache entries
(host code only; it calls libfav4_bshd.so, which it finds beside itself).
"""
from __future__ import annotations

import argparse
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parents[1]
REPO_ROOT = PKG_ROOT.parent
CSRC = PKG_ROOT / "csrc"
INCLUDE = REPO_ROOT / "include"
BUILD = PKG_ROOT / "build"
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-shared", "-Xptxas", "-v",
          f"-I{INCLUDE}", f"-I{CSRC}"]
TARGETS = {
    "libfav4_bshd.so": ["fav4_bshd.cu", "paged.cu"],
    "libfav4_probe.so": ["probe.cu"],
}
BINDING = "fav4_paged_torch.so"
BINDING_SRC = CSRC / "paged_torch.cpp"


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _stale(out: Path, deps) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _run(cmd, log: Path, name: str, verbose: bool) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    log.write_text(r.stdout + r.stderr)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"the compiler failed for {name}")
    if verbose:
        print(" ".join(cmd))


def _torch() -> str | None:
    """Which torch the binding is compiled against, without importing it; None where there is none with CUDA."""
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None or not (Path(spec.origin).parent / "lib" / "libc10_cuda.so").exists():
        return None
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:  # a source tree on the path
        version = "?"
    return f"{version} {spec.origin} python {sys.version.split()[0]}"


def binding_command(out: Path) -> list[str]:
    import sysconfig

    import torch

    home, lib = Path(nvcc()).resolve().parents[1], Path(torch.__file__).parent
    includes = [lib / "include", lib / "include" / "torch" / "csrc" / "api" / "include", home / "include",
                sysconfig.get_paths()["include"], INCLUDE]
    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    # -nostdlib++ and libstdc++.so: the C++ runtime that torch itself runs on, never a static copy of the compiler's
    return [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-nostdlib++",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *[f"-isystem{i}" for i in includes],
            str(BINDING_SRC), "-o", str(out), f"-L{BUILD}", f"-L{lib / 'lib'}", f"-L{home / 'lib64'}",
            "-l:libfav4_bshd.so", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-lcudart",
            "-l:libstdc++.so.6", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{lib / 'lib'}"]


def build(force: bool = False, verbose: bool = False) -> list[Path]:
    BUILD.mkdir(parents=True, exist_ok=True)
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    built = []
    for lib, srcs in TARGETS.items():
        out = BUILD / lib
        if force or _stale(out, deps):
            cmd = [nvcc(), *ARCH_FLAGS, *COMMON, "-o", str(out), *[str(CSRC / s) for s in srcs]]
            _run(cmd, BUILD / f"{lib}.ptxas.txt", lib, verbose)
        built.append(out)
    out, stamp, torch_now = BUILD / BINDING, BUILD / f"{BINDING}.torch", _torch()
    if torch_now is None:
        print(f"{BINDING} is not built: there is no torch with CUDA here (the C ABI does not need it)", file=sys.stderr)
        return built
    # it links against torch's C++ ABI: another torch needs another binding
    other = not stamp.exists() or stamp.read_text() != torch_now
    if force or other or _stale(out, [BINDING_SRC, *INCLUDE.glob("*.h")]):
        _run(binding_command(out), BUILD / f"{BINDING}.log", BINDING, verbose)
        stamp.write_text(torch_now)
    return [*built, out]


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    for p in build(force=a.force, verbose=True):
        print("built", p)


if __name__ == "__main__":
    main()
