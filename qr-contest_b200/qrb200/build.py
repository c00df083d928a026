"""Build ``libqrb200.so`` in-tree with nvcc for sm_100a (no GPU needed to compile).

    python -m qrb200.build            (from the qr-contest_b200 directory)

The library has no PyTorch dependency: ``csrc/qrb_api.cu`` (the factorization) and
``csrc/qrb_layer.cu`` (the layer operators) are compiled to objects side by side and linked with
the CUDA runtime linked statically.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent                      # qr-contest_b200/
CSRC = ROOT / "csrc"
INCLUDE = ROOT.parent / "include"
LIB = PKG / "libqrb200.so"
TESTKIT = PKG / "libqrb200_testkit.so"   # single-stage entry points for the GPU unit tests
CHECKED = PKG / "libqrb200_checked.so"   # the library with the pivot-map bounds checks
NOWAIT = PKG / "libqrb200_nowait.so"     # the layer operators with bounded waits that run out at once

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
         "--expt-relaxed-constexpr", "-Xptxas", "-O3"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def up_to_date(target: Path, inputs) -> bool:
    if not target.exists():
        return False
    t = target.stat().st_mtime
    return all(p.exists() and p.stat().st_mtime <= t for p in inputs)


OBJ = ROOT / "build"                   # objects and their dependency files (git-ignored)


def _object(src: Path, defs) -> Path:
    return OBJ / (src.stem + "".join(d.replace("-D", "-").replace("=", "-") for d in defs) + ".o")


def _inputs(obj: Path):
    """The files an object was compiled from, as nvcc listed them (none: never compiled)."""
    dep = obj.with_suffix(".d")
    if not dep.exists():
        return None
    files = dep.read_text().replace("\\\n", " ").split(":", 1)[1].split()
    return [Path(f) for f in files if not f.startswith(("/usr", "/opt"))]


def _compile(src: Path, obj: Path, verbose: bool, extra) -> None:
    OBJ.mkdir(exist_ok=True)
    cmd = [nvcc(), *ARCH, *FLAGS, *extra, "-I", str(INCLUDE), "-MD", "-MF",
           str(obj.with_suffix(".d")), "-c", "-o", str(obj), str(src)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def _link(objs, out: Path, verbose: bool) -> None:
    cmd = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", str(out), *map(str, objs)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


OPS = PKG / "libqrb200_torch_ops.so"  # torch.ops.qrb200.* (links libqrb200.so)
PY = PKG / "_layers.so"               # the layer operators' Python functions (links OPS)


def _compile_host(src: Path, out: Path, verbose: bool, include, link) -> None:
    """A library against torch's headers and libraries, next to the ones it is linked to (rpath
    $ORIGIN).  No CUDA code is compiled here."""
    import torch
    from torch.utils import cpp_extension as ce
    cuda_home = Path(ce.CUDA_HOME or "/usr/local/cuda")
    abi = int(torch.compiled_with_cxx11_abi())
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           "-I", str(INCLUDE), "-I", str(cuda_home / "include"), *include]
    for d in ce.include_paths():
        cmd += ["-I", d]
    cmd += ["-o", str(out), str(src), "-L", str(PKG), "-Wl,-rpath,$ORIGIN"]
    for d in ce.library_paths():
        cmd += ["-L", d, f"-Wl,-rpath,{d}"]
    cmd += [*link, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def _compile_ops(verbose: bool) -> None:
    """The TORCH_LIBRARY operator library, linked to libqrb200.so."""
    _compile_host(CSRC / "qrb_torch_op.cpp", OPS, verbose, [], ["-l:libqrb200.so"])


def _compile_py(verbose: bool) -> None:
    """The Python module of the layer operators, linked to the operator library."""
    import sysconfig
    _compile_host(CSRC / "qrb_py_layers.cpp", PY, verbose, ["-I", sysconfig.get_paths()["include"]],
                  ["-l:libqrb200_torch_ops.so", "-ltorch_python"])


# what each library is linked from: (source, definitions)
_CHECK = ["-DQRB_BOUNDS_CHECK"]
_LINKS = ((LIB, [("qrb_api.cu", []), ("qrb_layer.cu", [])]),
          (CHECKED, [("qrb_api.cu", _CHECK), ("qrb_layer.cu", [])]),
          (TESTKIT, [("qrb_testkit.cu", ["-DQRB_PANEL_TIMERS"])]),
          (NOWAIT, [("qrb_api.cu", []), ("qrb_layer.cu", ["-DQRB_LAYER_WAIT_LIMIT=0"])]))


def build(force: bool = False, verbose: bool = False, extra=()) -> Path:
    # the nvcc runs are independent (minutes each): run them side by side
    from concurrent.futures import ThreadPoolExecutor
    jobs = {}
    for _, units in _LINKS:
        for name, defs in units:
            obj = _object(CSRC / name, defs)
            inputs = _inputs(obj)
            if force or inputs is None or not up_to_date(obj, inputs):
                jobs[obj] = (CSRC / name, obj, verbose, [*extra, *defs])
    with ThreadPoolExecutor(max_workers=max(1, len(jobs))) as ex:
        for f in [ex.submit(_compile, *job) for job in jobs.values()]:
            f.result()
    for out, units in _LINKS:
        objs = [_object(CSRC / name, defs) for name, defs in units]
        if force or not up_to_date(out, objs):
            _link(objs, out, verbose)
    if force or not up_to_date(OPS, [CSRC / "qrb_torch_op.cpp", CSRC / "qrb_torch_layers.h", *INCLUDE.glob("*.h")]):
        _compile_ops(verbose)
    if force or not up_to_date(PY, [CSRC / "qrb_py_layers.cpp", CSRC / "qrb_torch_layers.h", OPS]):
        _compile_py(verbose)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True,
          extra=["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else [])
