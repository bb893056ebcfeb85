"""Build libfme_cuda.so in-tree with nvcc for sm_100a (B200).

    python fast-mario-env_b200/build.py          # or __graft_entry__.build()

The library is a plain C-ABI shared object (no Python extension, no JIT). Each source is compiled to an object of its
own, side by side, and the objects are linked. FMA contraction is disabled for the env engine so that the INTER_AREA
float arithmetic keeps OpenCV's exact operation order; the operators of the memory policy are compiled with it.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libfme_cuda.so")
SOURCES = {"fme.cu": ["--fmad=false"], "fme_attn.cu": [], "fme_norm.cu": []}   # source: flags of its own
DEPS = ["fme.cu", "fme_kernels.cuh", "fme_core.h", "fme_agent.h", "fme_render.h", "fme_defs.h", "fme_tables.h", "fme_fast.h", "fme_dp.h", "fme_ppo.cuh", "fme_replay.cuh",
        "fme_host.h", "fme_mma.cuh", "fme_attn.cu", "fme_norm.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC)")


def commands(obj_dir: str, out: str = LIB, extra=()) -> tuple[list[list[str]], list[str]]:
    """The compile commands, one for each source, and the link command."""
    inc = os.path.join(os.path.dirname(HERE), "include")
    objs = [os.path.join(obj_dir, s.replace(".cu", ".o")) for s in SOURCES]
    compiles = [[nvcc_path(), *ARCH, "-O3", "-lineinfo", "-std=c++17", *flags, "-Xptxas", "-v", "-Xcompiler", "-fPIC",
                 "-I", inc, "-I", CSRC, *extra, "-c", os.path.join(CSRC, s), "-o", o]
                for (s, flags), o in zip(SOURCES.items(), objs)]
    return compiles, [nvcc_path(), *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", out]


def up_to_date(out: str = LIB) -> bool:
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    deps = [os.path.join(CSRC, d) for d in DEPS] + [os.path.join(os.path.dirname(HERE), "include", "fme.h")]
    return all(os.path.getmtime(d) <= t for d in deps if os.path.exists(d))


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    with tempfile.TemporaryDirectory() as obj_dir:
        compiles, link = commands(obj_dir)
        procs = [subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for c in compiles]
        said = [p.communicate()[0] for p in procs]
        for p, text in zip(procs, said):
            if p.returncode != 0:
                sys.stderr.write(text)
                raise RuntimeError("nvcc failed building libfme_cuda.so")
        r = subprocess.run(link, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("nvcc failed linking libfme_cuda.so")
    if verbose:
        sys.stderr.write("".join(said))
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
