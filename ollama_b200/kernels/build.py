"""Build the sm_100a kernel library in-tree with nvcc.

``python -m ollama_b200.kernels.build`` compiles every ``.cu`` of this directory for
``compute_100a / sm_100a`` and links ``libb200ops.so`` next to the sources (and the C++ host
helpers of ``ollama_b200/native`` into ``libb200host.so``).  Objects are rebuilt only when their
source (or a header) is newer.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import hashlib
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
NATIVE = os.path.join(os.path.dirname(HERE), "native")
LIB = os.path.join(HERE, "libb200ops.so")
HOSTLIB = os.path.join(NATIVE, "libb200host.so")
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "--expt-relaxed-constexpr",
              "-Xcompiler", "-fPIC,-fvisibility=hidden"]


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


# sources of a part of the library, for a first start that should compile what one kind of model needs and no more
GROUPS = {"stack": ("attn_decode_mma.cu", "attn_latent.cu", "attn_paged.cu", "attn_pages8.cu", "attn_pages8_tc.cu", "attn_prefill_tc.cu", "depth.cu", "elementwise.cu", "gemm_f32.cu", "gemm_tc.cu", "gemv_rows.cu",
                    "gru.cu", "latent.cu", "moe.cu", "moe_rows.cu", "norm_rows.cu", "pages8.cu", "sample.cu", "ssd.cu", "ssd_chunk.cu", "ssm.cu")}


# modules of calls (ops/<name>_call.cpp) and the kernel source that says which argument blocks (<name>_args.h) the library takes
CALLS = {"pages8": "pages8.cu", "kv4": "kv4.cu"}


def build_group(group: str, verbose: bool = False, force: bool = False) -> str:
    """Compile the sources of ``group`` and link them into a library of their own; their objects are the ones a later full build uses."""
    lib = os.path.join(HERE, f"libb200{group}.so")
    _compile(sorted(GROUPS[group]), lib, verbose, force)
    if "pages8.cu" in GROUPS[group]:
        build_calls(verbose, force)
    return lib


def build(verbose: bool = False, force: bool = False) -> str:
    _compile(sorted(f for f in os.listdir(HERE) if f.endswith(".cu")), LIB, verbose, force)
    build_host(verbose, force)
    for what in CALLS:
        build_calls(verbose, force, what)
    return LIB


def _compile(srcs: list[str], lib: str, verbose: bool, force: bool) -> None:
    nvcc = _nvcc()
    hdrs = [os.path.join(HERE, f) for f in os.listdir(HERE) if f.endswith((".cuh", ".h"))]
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    jobs = []
    for s in srcs:
        src, obj = os.path.join(HERE, s), os.path.join(objdir, s[:-3] + ".o")
        if force or _stale(obj, [src] + hdrs):
            cmd = [nvcc, *NVCC_FLAGS, *(_layout_flag(n) for n, of in CALLS.items() if of == s), "-c", src, "-o", obj] + (["-Xptxas", "-v"] if verbose else [])
            jobs.append((s, cmd))

    def run(job):
        name, cmd = job
        r = subprocess.run(cmd, capture_output=True, text=True)
        return name, r.returncode, r.stdout + r.stderr

    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            for name, rc, out in ex.map(run, jobs):
                if verbose or rc:
                    sys.stderr.write(f"--- {name}\n{out}\n")
                if rc:
                    raise RuntimeError(f"nvcc failed on {name}")
    objs = [os.path.join(objdir, s[:-3] + ".o") for s in srcs]
    if force or _stale(lib, objs):
        part = f"{lib}.{os.getpid()}"          # linked beside it and renamed: another process never loads half a library
        r = subprocess.run([nvcc, "-shared", "-o", part, *objs, "-lcuda"], capture_output=True, text=True)
        if r.returncode:
            raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
        os.replace(part, lib)


def build_host(verbose: bool = False, force: bool = False) -> str | None:
    """C++ host-side helpers (no CUDA needed): device query, BPE merge loop, GGUF block codecs."""
    if not os.path.isdir(NATIVE):
        return None
    srcs = sorted(os.path.join(NATIVE, f) for f in os.listdir(NATIVE) if f.endswith(".cpp"))
    if not srcs:
        return None
    if force or _stale(HOSTLIB, srcs):
        cmd = ["g++", "-O2", "-std=c++17", "-ffp-contract=off", "-shared", "-fPIC", "-fvisibility=hidden", "-o", HOSTLIB, *srcs, "-ldl", "-lpthread"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or r.returncode:
            sys.stderr.write(r.stdout + r.stderr)
        if r.returncode:
            raise RuntimeError("host library build failed")
    probe_src, probe_bin = os.path.join(NATIVE, "devquery.cpp"), os.path.join(NATIVE, "devquery")
    if os.path.exists(probe_src) and (force or _stale(probe_bin, [probe_src])):      # the device probe also exists as a stand-alone child program
        r = subprocess.run(["g++", "-O2", "-std=c++17", "-DB2_DEVQUERY_MAIN", probe_src, "-ldl", "-o", probe_bin], capture_output=True, text=True)
        if r.returncode:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("device probe build failed")
    return HOSTLIB


def _text(*path: str) -> bytes:
    with open(os.path.join(*path), "rb") as f:
        return f.read()


def _layout_flag(what: str = "pages8") -> str:
    """What the kernel library and a module of calls are both compiled with: a number that follows from the argument blocks that they share."""
    return f"-D{what.upper()}_LAYOUT=0x{hashlib.sha256(_text(HERE, f'{what}_args.h')).hexdigest()[:16]}ull"


def calls_path(what: str = "pages8") -> str:
    """A module of calls for this Python and torch, of the sources as they are: one that was built for others, or from others, has another name."""
    import torch
    ops = os.path.join(os.path.dirname(HERE), "ops")
    made_from = hashlib.sha256(_text(ops, f"{what}_call.cpp") + _text(ops, "call_args.h") + _text(HERE, f"{what}_args.h")).hexdigest()[:12]
    return os.path.join(ops, f"_{what}.{sys.implementation.cache_tag}-torch{torch.__version__}.{made_from}.so")


def build_calls(verbose: bool = False, force: bool = False, what: str = "pages8") -> str:
    """A Python module of calls whose arguments are checked in C++ (ops/<what>_call.cpp); needs torch's headers, no GPU."""
    src, out = os.path.join(os.path.dirname(HERE), "ops", f"{what}_call.cpp"), calls_path(what)
    if force or not os.path.exists(out):
        import sysconfig

        from torch.utils.cpp_extension import include_paths, library_paths
        cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
        part = f"{out}.{os.getpid()}"
        cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", _layout_flag(what), *(f"-I{d}" for d in (*include_paths(), os.path.join(cuda, "include"), sysconfig.get_paths()["include"])),
               "-o", part, src, *(f"-L{d}" for d in (*library_paths(), os.path.join(cuda, "lib64"))), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or r.returncode:
            sys.stderr.write(r.stdout + r.stderr)
        if r.returncode:
            raise RuntimeError(f"g++ failed on {what}_call.cpp")
        os.replace(part, out)
        for old in glob.glob(glob.escape(out.rsplit(".", 2)[0]) + ".*.so"):          # of the same Python and torch
            if old != out:
                os.remove(old)
    return out


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
