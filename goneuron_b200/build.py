"""Builds libgoneuron_cuda.so in-tree with nvcc for sm_100a (cross-compiles without a GPU)."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
SO = os.path.join(HERE, "libgoneuron_cuda.so")
UNITS = ["model.cu", "operators.cu"]          # compiled side by side
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "-Xcompiler", "-fPIC", "-diag-suppress", "177,550"]


def sources():
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh"))] + \
           [os.path.join(os.path.dirname(HERE), "include", "goneuron_cuda.h")]


def up_to_date():
    return os.path.exists(SO) and all(os.path.getmtime(SO) >= os.path.getmtime(s) for s in sources())


def _object(unit):
    return os.path.join(CSRC, unit[:-3] + ".o")


def _depends(unit):
    """The files that the unit's object was made from, as nvcc listed them; None if there is no object yet."""
    try:
        with open(_object(unit) + ".d") as f:
            return f.read().split(":", 1)[1].replace("\\\n", " ").split()
    except (OSError, IndexError):
        return None


def _object_up_to_date(unit):
    o, files = _object(unit), _depends(unit)
    return files is not None and os.path.exists(o) and all(os.path.exists(f) and os.path.getmtime(o) >= os.path.getmtime(f) for f in files)


def build(force=False, verbose=False):
    if not force and up_to_date():
        return SO
    jobs = []
    for u in UNITS:
        if force or not _object_up_to_date(u):
            cmd = [NVCC] + FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-MD", "-MF", _object(u) + ".d", "-c", "-o", _object(u), os.path.join(CSRC, u)]
            jobs.append((cmd, subprocess.Popen(cmd)))
    for cmd, p in jobs:
        p.wait()
    for cmd, p in jobs:
        if p.returncode:
            raise subprocess.CalledProcessError(p.returncode, cmd)
    subprocess.check_call([NVCC] + FLAGS + ["-shared", "-o", SO] + [_object(u) for u in UNITS] + ["-lcudart", "-ldl"])
    return SO


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(SO)
