"""Build libqwen35_fp8_hip.so (gfx950) from csrc/*.hip with hipcc.

Replaces the reference's compile.bat (nvcc -> two Windows DLLs): one shared
library exporting both the reference's ctypes symbols and the native qh_*
entry points.  Objects are compiled in parallel; the library is written next
to this file so it travels with the source tree, as are the extension modules
_paged_host.so and _serve_host.so (csrc/*_host.cpp, host code against torch's
headers).  The library needs hipcc alone: it is linked whether the modules
build or not, and where there is no torch they are left out.

    python build.py [--jobs N] [--debug]
"""
import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_NAME = "libqwen35_fp8_hip.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
HOST_PATH = os.path.join(HERE, "_paged_host.so")
ARCH = os.environ.get("QH_OFFLOAD_ARCH", "gfx950")

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-fvisibility=hidden",
    "-Wall",
    "-Wno-unused-result",
    # No packed-FP32 VALU ops anywhere in this library.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def hipcc():
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def compile_one(cc, src, obj, extra):
    cmd = [cc, *HIPCC_FLAGS, *extra, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {os.path.basename(src)}:\n{r.stderr}")
    return obj


def build_host(name, path, extra):
    """An extension module that checks and launches calls, csrc/`name`.cpp: its path, or None
    without a torch to build it against."""
    try:
        import torch
    except ImportError:
        return None
    root = os.path.dirname(torch.__file__)
    tmp = path + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-Wall", *extra,
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", os.path.join(root, "include"),
           "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I", sysconfig.get_paths()["include"], os.path.join(CSRC, name + ".cpp"), "-o", tmp,
           "-L", os.path.join(root, "lib"), "-lc10", "-ltorch_cpu", "-ltorch_python"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"{name}.cpp failed: {e}") from e
    if r.returncode != 0:
        raise RuntimeError(f"{name}.cpp failed:\n{r.stderr}")
    os.replace(tmp, path)
    return path


def build(jobs=None, debug=False, verbose=True):
    cc = hipcc()
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    extra = ["-g"] if debug else []
    srcs = sources()
    objs = [os.path.join(objdir, os.path.basename(s)[:-4] + ".o") for s in srcs]
    jobs = jobs or min(len(srcs), max(1, (os.cpu_count() or 4)))
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        hosts = [ex.submit(build_host, "paged_host", HOST_PATH, extra),
                 ex.submit(build_host, "serve_host", os.path.join(HERE, "_serve_host.so"), extra)]
        futs = [ex.submit(compile_one, cc, s, o, extra) for s, o in zip(srcs, objs)]
        for f in futs:
            f.result()
    tmp = LIB_PATH + ".tmp"
    # -z defs: an unresolved symbol (e.g. a kernel launch stub the host pass
    # failed to emit) fails the link instead of the first dlopen
    cmd = [cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-Wl,-z,defs", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB_PATH)
    if verbose:
        print(f"built {LIB_PATH} ({len(srcs)} sources, {ARCH})")
    if None in [h.result() for h in hosts] and verbose:
        print("no torch: without _paged_host.so and _serve_host.so, which paged.py, tables.py, adapters.py and "
              "sampling.py need")
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=None)
    ap.add_argument("--debug", action="store_true")
    a = ap.parse_args()
    try:
        build(a.jobs, a.debug)
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
