"""Builds libgoneuron_cuda.so in-tree with nvcc for sm_100a (cross-compiles without a GPU), and where torch is installed the module through which its tensors reach the
operators on device memory."""
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include", "goneuron_cuda.h")
SO = os.path.join(HERE, "libgoneuron_cuda.so")
TORCH_SO = os.path.join(HERE, "_torch_operators.so")
UNITS = ["model.cu", "operators.cu"]          # compiled side by side
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = os.environ.get("CXX", "g++")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "-Xcompiler", "-fPIC", "-diag-suppress", "177,550"]


def sources():
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh"))] + [INCLUDE]


def _newer(target, files):
    return os.path.exists(target) and all(os.path.exists(f) and os.path.getmtime(target) >= os.path.getmtime(f) for f in files)


def _torch():
    """Where torch is installed, without importing it; None if it is not."""
    spec = importlib.util.find_spec("torch")
    return os.path.dirname(spec.origin) if spec and spec.origin else None


def _torch_sources():
    return [os.path.join(CSRC, "torch_operators.cpp"), INCLUDE, os.path.join(_torch(), "version.py")]


def up_to_date():
    return _newer(SO, sources()) and (_torch() is None or _newer(TORCH_SO, _torch_sources()))


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
    files = _depends(unit)
    return files is not None and _newer(_object(unit), files)


def _torch_command():
    t = _torch()
    include = [os.path.join(t, "include"), os.path.join(t, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
               os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")]
    return [CXX, "-O2", "-std=c++17", "-fPIC", "-shared"] + [a for p in include for a in ("-isystem", p)] + \
           ["-o", TORCH_SO, os.path.join(CSRC, "torch_operators.cpp"), "-L" + HERE, "-lgoneuron_cuda", "-Wl,-rpath,$ORIGIN",
            "-L" + os.path.join(t, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10"]


def _wait(jobs):
    for _, p in jobs:
        p.wait()
    for cmd, p in jobs:
        if p.returncode:
            raise subprocess.CalledProcessError(p.returncode, cmd)


def build(force=False, verbose=False):
    if not force and up_to_date():
        return SO
    if force or not _newer(SO, sources()):
        jobs = []
        for u in UNITS:
            if force or not _object_up_to_date(u):
                cmd = [NVCC] + FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-MD", "-MF", _object(u) + ".d", "-c", "-o", _object(u), os.path.join(CSRC, u)]
                jobs.append((cmd, subprocess.Popen(cmd)))
        _wait(jobs)
        subprocess.check_call([NVCC] + FLAGS + ["-shared", "-o", SO] + [_object(u) for u in UNITS] + ["-lcudart", "-ldl"])
    if _torch() is not None and (force or not _newer(TORCH_SO, _torch_sources())):
        cmd = _torch_command()
        _wait([(cmd, subprocess.Popen(cmd))])
    return SO


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(SO)
