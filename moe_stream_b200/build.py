"""Build libmoestream_cuda (shared, for ctypes / FFI callers, and static, for a Rust build.rs)
in-tree under moe_stream_b200/_build/ with nvcc for sm_100a, and, where torch is installed, the extension that reads
torch tensors.  Run: python -m moe_stream_b200.build"""
from __future__ import annotations

import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "_build")
SOURCES = ["kernels_dense.cu", "kernels_moe.cu", "kernels_moe_tc.cu", "kernels_prefill.cu", "kernels_prefill_attn.cu", "kernels_exact.cu", "kernels_sample.cu", "kernels_ssm.cu", "kernels_batch.cu",
           "kernels_qk_rope.cu", "kernels_prompt_attn.cu", "kernels_kv4.cu", "kernels_kv4_attn.cu", "runtime.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
         "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr"]
SO = os.path.join(OUT, "libmoestream_cuda.so")
A = os.path.join(OUT, "libmoestream_cuda.a")
BINDING = os.path.join(OUT, "_binding.so")
BINDING_TORCH = os.path.join(OUT, "_binding.torch")   # version.py of the torch that the extension was compiled against


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _text(path: str) -> str:
    if not os.path.exists(path):
        return ""
    with open(path) as f:
        return f.read()


def build(verbose: bool = False) -> str:
    os.makedirs(OUT, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    headers.append(os.path.join(os.path.dirname(HERE), "include", "moestream_cuda.h"))
    objs, cmds = [], []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(OUT, src.replace(".cu", ".o"))
        if _stale(o, [s] + headers):
            cmds.append([NVCC, *FLAGS, "-c", s, "-o", o])
        objs.append(o)
    src = os.path.join(CSRC, "binding.cpp")
    torch, version = importlib.util.find_spec("torch"), None   # found, not imported: the library itself needs none
    if torch is None:
        print("torch is not installed: the library is built without the extension for torch tensors", file=sys.stderr)
    else:
        at = os.path.dirname(torch.origin)
        version = _text(os.path.join(at, "version.py"))
        if _stale(BINDING, [src, headers[-1]]) or _text(BINDING_TORCH) != version:
            for old in (BINDING, BINDING_TORCH):
                if os.path.exists(old):
                    os.remove(old)
            cmds.append(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-isystem", os.path.join(at, "include"),
                         "-I" + sysconfig.get_paths()["include"], src, "-o", BINDING, "-L" + os.path.join(at, "lib"), "-lc10",
                         "-ltorch_cpu", "-ltorch_python"])
    # translation units compile in parallel (one compiler process each)
    procs = []
    for cmd in cmds:
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        procs.append((cmd, subprocess.Popen(cmd)))
    failed = [cmd for cmd, p in procs if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    if version is not None and _text(BINDING_TORCH) != version:
        with open(BINDING_TORCH, "w") as f:
            f.write(version)
    if _stale(SO, objs):
        subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", SO, *objs,
                        "-Xcompiler", "-fPIC", "-lcuda"], check=True)
    if _stale(A, objs):
        if os.path.exists(A):
            os.remove(A)
        subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-lib", "-o", A, *objs], check=True)
    return SO


if __name__ == "__main__":
    print(build(verbose=True))
