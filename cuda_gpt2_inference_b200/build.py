"""Build recipe for the CUDA library (in-tree, sm_100a).

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` (``-gencode
arch=compute_100a,code=sm_100a -lineinfo -O3 --use_fast_math``) into
``cuda_gpt2_inference_b200/libgpt2b.so``.  ``--use_fast_math`` matches the
reference build (Makefile:137) so fast-math divisions in the quantisers give
the reference's bytes.  Objects go to ``cuda_gpt2_inference_b200/_build/``.
``csrc/bind.cpp`` (operators on torch tensors without ctypes) becomes
``cuda_gpt2_inference_b200/_bind.so``, against the headers of the installed torch, and is
built again when torch or Python changes.  The library is linked whatever becomes of it, and it is left out,
with a message, where torch, g++ or Python's headers are absent: C and C++ callers need none of them.

Usage: ``python -m cuda_gpt2_inference_b200.build [--force] [--verbose] [--trace]``.
``--trace`` builds ``libgpt2b_trace.so`` instead (objects in ``_build_trace/``): the
persistent kernel stamps ``%globaltimer`` at its phase boundaries
(``GPT2B_PERSIST_TRACE``; ``bench.py --profile-case trace`` reads them).  Load it with
``GPT2B_LIB=<path>``.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libgpt2b.so")
BIND = os.path.join(HERE, "_bind.so")
BIND_FOR = os.path.join(OBJ, "bind_for.txt")  # the torch and Python that _bind.so was built against
OBJ_TRACE = os.path.join(HERE, "_build_trace")
LIB_TRACE = os.path.join(HERE, "libgpt2b_trace.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")
NVCC = os.path.join(CUDA_HOME, "bin", "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "--use_fast_math", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-fvisibility=default",
              f"-I{INCLUDE}", f"-I{CSRC}"]


def _nccl_paths():
    """Include and library directories of the NCCL shipped with torch's wheels."""
    try:
        import nvidia.nccl  # type: ignore
        base = os.path.dirname(nvidia.nccl.__file__) if nvidia.nccl.__file__ else list(nvidia.nccl.__path__)[0]
    except Exception:  # pragma: no cover - probed at build time
        return None, None
    inc, lib = os.path.join(base, "include"), os.path.join(base, "lib")
    if os.path.exists(os.path.join(inc, "nccl.h")) and os.path.exists(os.path.join(lib, "libnccl.so.2")):
        return inc, lib
    return None, None


def _run(cmd, verbose=False):
    if verbose:
        print(" ".join(cmd))
    p = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if p.returncode != 0:
        raise RuntimeError(os.path.basename(cmd[0]) + " failed:\n" + " ".join(cmd) + "\n" + p.stdout[-6000:])
    return p.stdout


def _headers():
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(INCLUDE, "*.h"))


def _bind_missing():
    """What keeps the binding from being built here, or None."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        return "torch"
    if not os.path.exists(os.path.join(spec.submodule_search_locations[0], "include", "ATen", "core", "Tensor.h")):
        return "torch's headers"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python's headers"
    return None if shutil.which("g++") else "g++"


def _bind_for():
    try:
        torch = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        torch = "?"
    return f"torch {torch} in {importlib.util.find_spec('torch').submodule_search_locations[0]}, Python {sys.version}"


def _bind_command():
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    libs = os.path.join(torch, "lib")
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", f"-I{INCLUDE}",
            f"-I{sysconfig.get_paths()['include']}", f"-I{torch}/include", f"-I{torch}/include/torch/csrc/api/include",
            f"-I{CUDA_HOME}/include", os.path.join(CSRC, "bind.cpp"), "-o", BIND, f"-L{libs}", "-ltorch_python",
            "-ltorch_cpu", "-lc10_cuda", "-lc10", f"-Wl,-rpath,{libs}"]


def build_binding(force: bool = False, verbose: bool = False) -> bool:
    """Compile csrc/bind.cpp into _bind.so where it is out of date; False (and a message) where that cannot be done."""
    missing = _bind_missing()
    if missing:
        print(f"{os.path.basename(BIND)} left out: no {missing} here; the operators for batches on torch tensors "
              "(ops.py) need it, the C ABI does not", file=sys.stderr)
        return False
    made_for = open(BIND_FOR).read() if os.path.exists(BIND_FOR) else ""
    sources = [os.path.join(CSRC, "bind.cpp"), os.path.join(INCLUDE, "gpt2_b200.h"), __file__]
    if force or not os.path.exists(BIND) or made_for != _bind_for() or \
            os.path.getmtime(BIND) < max(os.path.getmtime(f) for f in sources):
        _run(_bind_command(), verbose)
        os.makedirs(os.path.dirname(BIND_FOR), exist_ok=True)
        with open(BIND_FOR, "w") as f:
            f.write(_bind_for())
    return True


def build(force: bool = False, verbose: bool = False, jobs: int | None = None, ptxas_info: bool = False,
          trace: bool = False) -> str:
    """Compile csrc/*.cu into libgpt2b.so (or the trace build) and _bind.so, incrementally; returns the library's path."""
    obj_dir, lib = (OBJ_TRACE, LIB_TRACE) if trace else (OBJ, LIB)
    os.makedirs(obj_dir, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdr_t = max((os.path.getmtime(h) for h in _headers()), default=0.0)
    nccl_inc, nccl_lib = _nccl_paths()
    extra = [f"-I{nccl_inc}", "-DGPT2B_HAVE_NCCL=1"] if nccl_inc else []
    if trace:
        extra.append("-DGPT2B_PERSIST_TRACE=1")
    objs, work = [], []
    for s in srcs:
        o = os.path.join(obj_dir, os.path.basename(s)[:-3] + ".o")
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr_t,
                                                                         os.path.getmtime(__file__)):
            cmd = [NVCC, *ARCH, *NVCC_FLAGS, *extra, "-c", s, "-o", o]
            if ptxas_info:
                cmd.insert(1, "-Xptxas=-v")
            work.append(cmd)
    with cf.ThreadPoolExecutor(max_workers=jobs or os.cpu_count() or 4) as ex:
        binding = None if trace else ex.submit(build_binding, force, verbose)
        outs = list(ex.map(lambda c: _run(c, verbose), work))
        if ptxas_info:
            for o in outs:
                print(o)
        if force or not os.path.exists(lib) or any(os.path.getmtime(lib) < os.path.getmtime(o) for o in objs):
            link = [NVCC, *ARCH, "-shared", "-o", lib, *objs, "-lcudart"]
            if nccl_lib:
                link += [f"-L{nccl_lib}", "-l:libnccl.so.2", f"-Xlinker=-rpath,{nccl_lib}"]
            _run(link, verbose)
        if binding:
            binding.result()  # an error of its compiler comes after the library is there
    return lib


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true", help="print -Xptxas -v register/spill/smem usage")
    ap.add_argument("--trace", action="store_true", help="build libgpt2b_trace.so (persistent-kernel phase stamps)")
    a = ap.parse_args()
    print(build(a.force, a.verbose, ptxas_info=a.ptxas_info, trace=a.trace))
    return 0


if __name__ == "__main__":
    sys.exit(main())
