"""Build libxp_cuda.so in-tree with nvcc for sm_100a (and the test oracles).

    python -m xpose_b200.build
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libxp_cuda.so")
OBJ = os.path.join(HERE, "build")
# one translation unit each, compiled side by side and linked into the library
UNITS = [os.path.join(HERE, "csrc", f) for f in ("xp_cuda.cu", "serving.cu")]
# torch tensors to the serving calls (CPython extension, linked to the library)
BINDING = os.path.join(HERE, "csrc", "serving_torch.cpp")
BINDING_LIB = os.path.join(HERE, "_serving.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else "nvcc")

NVCC_FLAGS = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC",
    "-diag-suppress", "1886,842",
]


def _sources():
    d = os.path.join(HERE, "csrc")
    return [os.path.join(d, f) for f in os.listdir(d)] + [os.path.join(ROOT, "include", "xp_cuda.h")]


def _stale(out, srcs):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(not os.path.exists(s) or os.path.getmtime(s) > t for s in srcs)


def _includes(obj, unit):
    """The files an object was made from, by the dependency file beside it."""
    dep = obj + ".d"
    if not os.path.exists(dep):
        return _sources()
    words = open(dep).read().replace("\\\n", " ").split(":", 1)[1].split()
    return [unit] + [w for w in words if os.path.realpath(w).startswith(ROOT + os.sep)]


def build_cuda(force=False, verbose=False):
    if not force and not _stale(LIB, _sources()):
        return LIB
    os.makedirs(OBJ, exist_ok=True)

    def compile_unit(unit):
        obj = os.path.join(OBJ, os.path.basename(unit) + ".o")
        if force or _stale(obj, _includes(obj, unit)):
            cmd = [NVCC, *NVCC_FLAGS, "-MD", "-MF", obj + ".d", "-c", "-o", obj, unit]
            if verbose:
                print(" ".join(cmd))
            subprocess.run(cmd, check=True)
        return obj

    with ThreadPoolExecutor(len(UNITS)) as pool:
        objs = list(pool.map(compile_unit, UNITS))
    subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", LIB, *objs], check=True)
    return LIB


def build_binding(force=False, verbose=False):
    if not force and not _stale(BINDING_LIB, [BINDING, os.path.join(ROOT, "include", "xp_cuda.h")]):
        return BINDING_LIB
    import sysconfig

    from torch.utils.cpp_extension import include_paths, library_paths

    inc = [sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")]
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-o", BINDING_LIB, BINDING,
           *[f"-I{d}" for d in inc], *[x for d in include_paths() for x in ("-isystem", d)],
           "-L" + HERE, "-lxp_cuda", "-Wl,-rpath,$ORIGIN",
           *[f"-L{d}" for d in library_paths()], "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    return BINDING_LIB


def build_oracle(verbose=False):
    """The CPU checkers (test infrastructure): oracle/liboracle.so always,
    oracle/_ref/libxpref.so when the reference tree is present."""
    env = dict(os.environ)
    env.pop("CC", None)
    env.pop("CXX", None)
    subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "oracle")], check=True, env=env,
                   stdout=None if verbose else subprocess.DEVNULL)


def main():
    build_cuda(force="--force" in sys.argv, verbose=True)
    build_binding(force="--force" in sys.argv, verbose=True)
    build_oracle(verbose=True)
    print("built", LIB)


if __name__ == "__main__":
    main()
