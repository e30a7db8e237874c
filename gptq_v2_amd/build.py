"""Builds gptq_v2_amd/lib/libgptq_amd.so (hipcc, gfx950 only) and the torch binding of the serving operators (g++).  Run as a
script, `python gptq_v2_amd/build.py`: importing the package needs the library this produces; the binding is needed by the
serving operators alone, and a failure to build it is raised when the library is there."""
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "lib", "libgptq_amd.so")
SOURCES = ["gq_core.hip", "xtx.hip", "hessian.hip", "sgemm.hip", "quantize.hip", "pack.hip", "w4a16.hip", "wq_stream.hip", "gemm_nt.hip", "elementwise.hip",
           "logprobs.hip", "kv_append.hip", "attention_paged.hip", "attention_prompt.hip"]
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-fno-fast-math",
         # no packed fp32 instructions: some of their forms have given wrong results now and then on this chip
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-Wall", "-Wno-unused-function"]


BINDING = os.path.join(HERE, "_serving_binding.so")
STAMP = os.path.join(OBJ, "serving_binding.stamp")   # what BINDING was built with


def _binding_cmd() -> list:
    """g++ line of the torch-facing binding (csrc/serving_binding.cpp); the C library itself needs no torch headers."""
    import sysconfig
    import torch
    base = os.path.dirname(torch.__file__)
    lib = os.path.join(base, "lib")
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-I" + os.path.join(ROOT, "include"),
            "-isystem", os.path.join(base, "include"), "-isystem", os.path.join(base, "include", "torch", "csrc", "api", "include"),
            "-isystem", "/opt/rocm/include", "-isystem", sysconfig.get_paths()["include"], "-Wall", os.path.join(CSRC, "serving_binding.cpp"), "-o", BINDING,
            "-L" + lib, "-Wl,-rpath," + lib, "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_hip"]


def _hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found")
    return exe


def _stale(out: str, deps) -> bool:
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def _binding_stamp(cmd) -> str:
    """The binding is compiled against torch's C++ headers and Python's: another of either wants another binding."""
    import sysconfig
    import torch
    return "\n".join([torch.__version__, str(sysconfig.get_config_var("SOABI")), *cmd])


def _binding_stale(stamp: str) -> bool:
    if not os.path.exists(STAMP) or open(STAMP).read() != stamp:
        return True
    return _stale(BINDING, [os.path.join(CSRC, "serving_binding.cpp"), os.path.join(ROOT, "include", "gptq_amd.h")])


def _build_binding(force: bool, run) -> None:
    cmd = _binding_cmd()
    stamp = _binding_stamp(cmd)
    if force or _binding_stale(stamp):
        run(cmd)
        with open(STAMP, "w") as f:
            f.write(stamp)


def build(force: bool = False, verbose: bool = True) -> str:
    os.makedirs(OBJ, exist_ok=True)
    os.makedirs(os.path.dirname(LIB), exist_ok=True)
    hipcc = _hipcc()
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    headers.append(os.path.join(ROOT, "include", "gptq_amd.h"))
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    objs = []
    jobs = []
    for s in srcs:
        src = os.path.join(CSRC, s)
        obj = os.path.join(OBJ, s.replace(".hip", ".o"))
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            jobs.append([hipcc, *FLAGS, "-c", src, "-o", obj])

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)

    with ThreadPoolExecutor(max_workers=min(8, len(jobs) + 1)) as ex:
        binding = ex.submit(_build_binding, force, run)
        list(ex.map(run, jobs))
        if jobs or force or _stale(LIB, objs):
            run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB, *objs])
        binding.result()
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
