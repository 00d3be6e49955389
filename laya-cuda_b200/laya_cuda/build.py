"""Builds liblaya_b200.so in-tree with nvcc for sm_100a (B200), and the Python extension _mx8.

    python -m laya_cuda.build            # from laya-cuda_b200/
"""
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
CSRC = PACKAGE.parent / "csrc"
INCLUDE = PACKAGE.parents[1] / "include"
TARGET = PACKAGE / "liblaya_b200.so"
SOURCES = [CSRC / "laya_b200.cu", CSRC / "mx8.cu"]
DEPENDS = SOURCES + sorted(CSRC.glob("*.cuh")) + [INCLUDE / "laya_b200.h"]
# Named for this Python's ABI, so that another one does not load it.
EXTENSION = PACKAGE / ("_mx8" + sysconfig.get_config_var("EXT_SUFFIX"))
EXTENSION_SOURCE = CSRC / "mx8_python.cpp"
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
         "-Xcompiler", "-fPIC", "-shared", "-cudart", "static", "--threads", "2"]


def nvcc():
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found")
    return found


def up_to_date(target, depends):
    if not target.exists():
        return False
    built = target.stat().st_mtime
    return all(p.stat().st_mtime <= built for p in depends)


def run(target, cmd, verbose):
    tmp = target.with_suffix(".so.tmp")
    cmd = [*cmd[:1], "-o", str(tmp), *cmd[1:]]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, target)


def build_extension(verbose=False):
    """_mx8, which laya_cuda.mx8 alone needs: without this Python's headers it is left out, and one built from older
    sources is taken away, so that importing laya_cuda.mx8 says so."""
    EXTENSION.with_name("_mx8.so").unlink(missing_ok=True)  # an earlier build's, which every Python would load
    include = Path(sysconfig.get_paths()["include"])
    if not (include / "Python.h").exists():
        EXTENSION.unlink(missing_ok=True)
        print(f"{EXTENSION.name} is not built, and laya_cuda.mx8 not available: no {include / 'Python.h'}", file=sys.stderr)
        return
    run(EXTENSION, [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
                    "-I", str(include), str(EXTENSION_SOURCE)], verbose)


def build(force=False, verbose=False):
    if force or not up_to_date(TARGET, DEPENDS):
        run(TARGET, [nvcc(), *FLAGS, "-I", str(INCLUDE), *map(str, SOURCES)], verbose)
    if force or not up_to_date(EXTENSION, [EXTENSION_SOURCE, INCLUDE / "laya_b200.h"]):
        build_extension(verbose)
    return TARGET


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
