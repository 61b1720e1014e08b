"""Compile the in-tree libraries with hipcc.

* ``libfsctep_hip.so``: the gfx950 HIP kernels behind the C ABI of ``include/fsctep.h``.
* ``libfsctep_torch.so``: the ``torch.ops.fsctep.*`` registration (schemas, device, Meta and
  autograd kernels) over that C ABI; loadable by LibTorch processes without Python.
* ``tests/cpp/core_run``: a LibTorch program with no Python that runs an exported core.pt the way the
  LAMMPS engine does (used by the GPU tests of the TorchScript core).

    python -m fsctep_amd.build
"""

from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libfsctep_hip.so")
TORCH_LIB = os.path.join(PKG, "libfsctep_torch.so")
CORE_RUN_SRC = os.path.join(ROOT, "tests", "cpp", "core_run.cpp")
CORE_RUN = os.path.join(ROOT, "tests", "cpp", "core_run")

HIP_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
    # packed fp32 (v_pk_*_f32) code generation disabled for every kernel
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def _torch_dirs() -> tuple[str, str]:
    import torch
    base = os.path.dirname(torch.__file__)
    return os.path.join(base, "include"), os.path.join(base, "lib")


def _check(proc, what: str) -> str:
    out, err = proc.communicate()
    if proc.returncode != 0:
        sys.stderr.write(out + err)
        raise RuntimeError(f"building {what} failed")
    return "\n".join(ln for ln in (out + err).splitlines()
                     if ln.strip() and "packed-fp32-ops" not in ln and "not a recognized feature" not in ln)


def build(verbose: bool = False) -> str:
    """Everything is made in a folder of its own, which goes whether the build succeeds or not; the libraries are put in place
    together at the end."""
    os.makedirs(os.path.join(PKG, "_build"), exist_ok=True)
    tmp = tempfile.mkdtemp(dir=os.path.join(PKG, "_build"))
    try:
        return _build(tmp, verbose)
    finally:
        shutil.rmtree(tmp)
        try:
            os.rmdir(os.path.dirname(tmp))
        except OSError:                      # another build's folder is there
            pass


def _build(tmp: str, verbose: bool) -> str:
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    inc = ["-I", os.path.join(ROOT, "include"), "-I", CSRC]
    lib, torch_lib, core_run = (os.path.join(tmp, os.path.basename(name)) for name in (LIB, TORCH_LIB, CORE_RUN))
    hip_srcs = sources()
    hip_objs = [os.path.join(tmp, os.path.basename(src) + ".o") for src in hip_srcs]
    hip_ccs = [[hipcc, *HIP_FLAGS, *inc, "-c", src, "-o", obj] for src, obj in zip(hip_srcs, hip_objs)]
    hip_link = [hipcc, *HIP_FLAGS, "-shared", "-Wl,-soname,libfsctep_hip.so", *hip_objs, "-o", lib]
    tinc, tlib = _torch_dirs()
    torch_srcs = ["torch_ops.cpp", "torch_bucket_ops.cpp", "torch_expert_ops.cpp", "torch_learn_ops.cpp"]
    objs = [os.path.join(tmp, src.replace(".cpp", ".o")) for src in torch_srcs]
    torch_ccs = [[hipcc, "-std=c++17", "-O2", "-fPIC", "-c", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
                  "-D_GLIBCXX_USE_CXX11_ABI=1", "-I", tinc, "-I", os.path.join(tinc, "torch", "csrc", "api", "include"),
                  "-I", "/opt/rocm/include", *inc, os.path.join(CSRC, src), "-o", obj]
                 for src, obj in zip(torch_srcs, objs)]
    core_cc = ["g++", "-std=c++17", "-O1", "-D_GLIBCXX_USE_CXX11_ABI=1", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
               "-I", tinc, "-I", os.path.join(tinc, "torch", "csrc", "api", "include"), "-I", "/opt/rocm/include",
               CORE_RUN_SRC, "-o", core_run,
               "-L", tlib, "-Wl,--no-as-needed", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip",
               f"-Wl,-rpath,{tlib}", "-L", "/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath,/opt/rocm/lib", "-ldl"]
    link = [hipcc, "-shared", "-fPIC", *objs, "-o", torch_lib, "-L", tmp, "-lfsctep_hip", "-L", tlib, "-ltorch",
            "-ltorch_cpu", "-lc10", "-lc10_hip", "-ltorch_hip", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{tlib}"]
    jobs = [*zip(hip_ccs, map(os.path.basename, hip_srcs)), *zip(torch_ccs, torch_srcs), (core_cc, "tests/cpp/core_run")]
    if verbose:
        print("\n".join(" ".join(c) for c in (*(c for c, _ in jobs), hip_link, link)), flush=True)

    def run(job):
        proc = subprocess.Popen(job[0], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
        return _check(proc, job[1])

    # the sources with the most kernels first: they take the longest
    jobs.sort(key=lambda job: -os.path.getsize(next(a for a in job[0] if a.endswith((".hip", ".cpp")))))
    with ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
        notes = list(pool.map(run, jobs))
    notes += [run((hip_link, "libfsctep_hip.so")), run((link, "libfsctep_torch.so"))]
    for made, place in ((lib, LIB), (torch_lib, TORCH_LIB), (core_run, CORE_RUN)):
        os.replace(made, place)
    if verbose and any(notes):
        print("\n".join(n for n in notes if n))
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
