"""Build the bpt CUDA library in-tree: kvq-decode_b200/bpt/libbpt_b200.so.

    python kvq-decode_b200/build.py [--force] [--verbose]

Compiles every ``csrc/*.cu`` for sm_100a only (``-gencode arch=compute_100a,code=sm_100a``)
with nvcc and links one shared library exporting the C ABI declared in ``include/bpt.h``, and
``csrc/bind.cpp`` with the host compiler against torch's headers as the extension module
``bpt/_bind`` (the Python binding of the scored decode and the eviction).
The CUDA runtime is linked statically; the driver API is reached through
``cudaGetDriverEntryPointByVersion`` so the library has no link-time libcuda dependency.
Rebuilds only when a source or header is newer than what was built, or torch (whose C++ ABI
``bpt/_bind`` is tied to) is another than it was built with.
"""
import argparse
import glob
import importlib.metadata
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OUT = os.path.join(PKG, "bpt", "libbpt_b200.so")
BIND_SRC = os.path.join(CSRC, "bind.cpp")
BIND_OUT = os.path.join(PKG, "bpt", "_bind" + sysconfig.get_config_var("EXT_SUFFIX"))
BIND_STAMP = os.path.join(PKG, "_build", "bind.torch")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3", "--expt-relaxed-constexpr",
         "-Xptxas", "-O3"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def deps():
    return (sources() + glob.glob(os.path.join(CSRC, "*.cuh")) +
            glob.glob(os.path.join(CSRC, "*.h")) +
            glob.glob(os.path.join(ROOT, "include", "*.h")) + [os.path.abspath(__file__)])


def newer(out, sources_) -> bool:
    """Whether ``out`` exists and no source is newer."""
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(d) <= t for d in sources_)


def up_to_date() -> bool:
    return newer(OUT, deps())


def bind_built_for() -> str:
    """The torch whose C++ ABI ``bpt/_bind`` is tied to."""
    return f"torch {importlib.metadata.version('torch')}\n"


def bind_up_to_date() -> bool:
    if not newer(BIND_OUT, [BIND_SRC, os.path.join(ROOT, "include", "bpt.h"),
                            os.path.abspath(__file__)]) or not os.path.exists(BIND_STAMP):
        return False
    with open(BIND_STAMP) as f:
        return f.read() == bind_built_for()


def start_bind(verbose: bool):
    """Compile and link ``bpt/_bind``; returns the running compiler."""
    import torch
    from torch.utils import cpp_extension
    inc = [os.path.join(ROOT, "include"), sysconfig.get_paths()["include"],
           *cpp_extension.include_paths(),
           os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           *[f"-isystem{i}" for i in inc], BIND_SRC, "-o", BIND_OUT + ".tmp", "-L" + libs,
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd))
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def build(force: bool = False, verbose: bool = False, extra=()) -> str:
    bind = None if not force and bind_up_to_date() else start_bind(verbose)
    if force or not up_to_date():
        build_library(verbose, extra)
    if bind is not None:
        out, _ = bind.communicate()
        if bind.returncode != 0:
            raise RuntimeError(f"{BIND_SRC} failed:\n{out}")
        os.replace(BIND_OUT + ".tmp", BIND_OUT)
        os.makedirs(os.path.dirname(BIND_STAMP), exist_ok=True)
        with open(BIND_STAMP, "w") as f:
            f.write(bind_built_for())
    return OUT


def build_library(verbose: bool, extra) -> None:
    objdir = os.path.join(PKG, "_build")
    os.makedirs(objdir, exist_ok=True)
    objs = []
    procs = []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        cmd = [nvcc(), *ARCH, *FLAGS, *extra, "-I", os.path.join(ROOT, "include"), "-c", src,
               "-o", obj]
        if verbose:
            print(" ".join(cmd))
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE,
                                            stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    failed = []
    for src, pr in procs:
        out, _ = pr.communicate()
        if pr.returncode != 0:
            failed.append((src, out))
        elif verbose and out.strip():
            print(out)
    if failed:
        msg = "\n".join(f"--- {s}\n{o}" for s, o in failed)
        raise RuntimeError("nvcc failed:\n" + msg)
    tmp = OUT + ".tmp"
    link = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", tmp, "-cudart",
            "static"]
    if verbose:
        print(" ".join(link))
    subprocess.run(link, check=True)
    os.replace(tmp, OUT)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-verbose", action="store_true",
                    help="print registers / spills / shared memory per kernel")
    a = ap.parse_args()
    extra = ["-Xptxas", "-v"] if a.ptxas_verbose else []
    print(build(force=a.force or a.ptxas_verbose, verbose=a.verbose or a.ptxas_verbose,
                extra=extra))


if __name__ == "__main__":
    sys.exit(main())
