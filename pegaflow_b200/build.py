"""Builds libpegaflow_b200.so (sm_100a kernels + C++ engine + C ABI) in-tree.

Every translation unit is compiled by nvcc for sm_100a only; the shared
library lands next to this file so it travels with the source tree.
The binding of the paged-cache operators for torch tensors (_kv_torch.so) is
compiled with the host compiler against the installed torch and this library;
where torch is not installed it is left out.
Run: python -m pegaflow_b200.build [--force]
"""

from __future__ import annotations

import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libpegaflow_b200.so"
TORCH_BINDING = PKG / "_kv_torch.so"
TORCH_STAMP = BUILD / "kv_torch.stamp"  # what the binding was built against

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC,-Wall,-Wno-unused-function",
    f"-I{ROOT / 'include'}",
    f"-I{CSRC}",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build pegaflow_b200")


def _sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")))


def _headers() -> list[Path]:
    return sorted(list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh")) + list((ROOT / "include").glob("*.h")))


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _torch_home() -> Path | None:
    """Where torch is installed: found, not imported, as the build needs its headers alone."""
    from importlib.util import find_spec

    try:
        spec = find_spec("torch")
    except ValueError:  # a stand-in of that name that was not imported from anywhere
        spec = None
    return Path(spec.origin).parent if spec and spec.origin else None


def _torch_stamp(home: Path) -> str:
    from importlib.metadata import PackageNotFoundError, version

    try:
        installed = version("torch")
    except PackageNotFoundError:  # a source tree on the path
        installed = "of no package"
    return f"{home}\ntorch {installed}\npython {sys.version}\n"


def _torch_command(src: Path, target: Path, torch: Path) -> list[str]:
    import sysconfig

    cuda = Path(nvcc()).resolve().parent.parent
    includes = [torch / "include", torch / "include/torch/csrc/api/include", sysconfig.get_paths()["include"],
                cuda / "include", ROOT / "include"]
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", *(f"-I{i}" for i in includes),
            str(src), "-o", str(target), f"-L{PKG}", "-lpegaflow_b200", f"-L{torch / 'lib'}", "-ltorch_python", "-ltorch",
            "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile and link the library if any source or header changed, and the
    torch binding if that or the installed torch did."""
    BUILD.mkdir(exist_ok=True)
    cc = nvcc()
    headers = _headers()
    jobs = []
    objs = []
    for src in _sources():
        obj = BUILD / (src.name + ".o")
        objs.append(obj)
        if force or _stale(obj, [src, *headers, Path(__file__)]):
            jobs.append([cc, *ARCH, *COMMON, "-c", str(src), "-o", str(obj)])

    def run(cmd: list[str]) -> None:
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
        if verbose and res.stderr.strip():
            print(res.stderr, flush=True)

    if jobs:
        with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
            list(ex.map(run, jobs))
    if force or jobs or _stale(LIB, objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [cc, *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-cudart", "static", "-lrt", "-lpthread"]
        run(cmd)
        os.replace(tmp, LIB)
    binding = CSRC / "torch" / "kv_binding.cpp"
    home = _torch_home()
    if home is None:
        if verbose:
            print("torch is not installed: the binding of the paged-cache operators is left out", flush=True)
        return LIB
    stamp = _torch_stamp(home)
    built_against = TORCH_STAMP.read_text() if TORCH_STAMP.exists() else None
    if force or built_against != stamp or _stale(TORCH_BINDING, [binding, ROOT / "include" / "pegaflow.h", Path(__file__)]):
        tmp = TORCH_BINDING.with_suffix(".so.tmp")
        run(_torch_command(binding, tmp, home))
        os.replace(tmp, TORCH_BINDING)
        TORCH_STAMP.write_text(stamp)
    return LIB


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args(argv)
    path = build(force=args.force, verbose=args.verbose)
    print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main())
