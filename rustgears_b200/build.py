"""Builds librg_npu.so (all CUDA kernels + the C ABI) in-tree for sm_100a, and the binding of
its serving entry points to torch tensors (_serving_bind.so) where a CUDA torch is installed."""
from __future__ import annotations

import glob
import os
import re
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "librg_npu.so")
BIND_SRC = os.path.join(HERE, "bind", "serving_bind.cpp")
BIND = os.path.join(HERE, "_serving_bind.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nccl_dirs():
    import importlib.util
    spec = importlib.util.find_spec("nvidia.nccl")
    if spec is None or not spec.submodule_search_locations:
        raise RuntimeError("NCCL (nvidia-nccl) not found")
    base = list(spec.submodule_search_locations)[0]
    return os.path.join(base, "include"), os.path.join(base, "lib")


def _flags():
    inc, _ = nccl_dirs()
    return ["-O3", "-std=c++17", "-lineinfo", "-fmad=false", "-Xcompiler", "-fPIC",
            "-Xcompiler", "-ffp-contract=off", "-Xptxas", "-v" if os.environ.get("RG_PTXAS_V") else "-O3",
            "-I", os.path.join(ROOT, "include"), "-I", inc]


def _compile(src: str) -> str:
    obj = os.path.join(OBJ, os.path.basename(src) + ".o")
    deps = [src] + glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        [os.path.join(ROOT, "include", "rg_npu.h")]
    if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(d) for d in deps):
        return obj
    cmd = [NVCC] + ARCH + _flags() + ["-c", src, "-o", obj]
    if src.endswith(".cpp"):
        cmd = [NVCC] + _flags() + ["-x", "c++", "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if os.environ.get("RG_PTXAS_V"):
        sys.stderr.write(r.stderr)
    return obj


def _torch_dir() -> str | None:
    """The installed torch's folder; None where there is none, or one without CUDA."""
    import importlib.util
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        return None
    torch = list(spec.submodule_search_locations)[0]
    return torch if os.path.exists(os.path.join(torch, "lib", "libtorch_cuda.so")) else None


def build_binding() -> str | None:
    """Compiles bind/serving_bind.cpp against torch's headers and links it to librg_npu.so, again
    when its source, the C header, torch or Python changed.  None without a CUDA torch: the
    library (C ABI, Rust crate, sessions) needs none, only rustgears_b200.serving does."""
    torch = _torch_dir()
    if torch is None:
        return None
    with open(os.path.join(torch, "version.py")) as f:
        text = f.read()
    version = re.search(r"""^__version__\s*=\s*['"]([^'"]+)""", text, flags=re.M)
    cuda = os.path.dirname(os.path.dirname(NVCC))
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-D_GLIBCXX_USE_CXX11_ABI=1",
           f'-DRG_TORCH_VERSION="{version.group(1) if version else "unknown"}"',
           "-I", os.path.join(ROOT, "include"), "-I", sysconfig.get_paths()["include"],
           "-I", os.path.join(torch, "include"), "-I", os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           "-I", os.path.join(cuda, "include"), BIND_SRC, "-o", BIND,
           "-L", os.path.join(torch, "lib"), "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10",
           "-L", HERE, "-l:librg_npu.so", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + os.path.join(torch, "lib")]
    built_for = "\n".join([sysconfig.get_config_var("SOABI") or sys.version, text] + cmd)
    header, key = os.path.join(ROOT, "include", "rg_npu.h"), os.path.join(OBJ, os.path.basename(BIND) + ".built_for")
    if os.path.exists(BIND) and os.path.getmtime(BIND) >= max(os.path.getmtime(f) for f in (BIND_SRC, header)) and \
            os.path.exists(key) and open(key).read() == built_for:
        return BIND
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"building {BIND} failed:\n{r.stdout}\n{r.stderr}")
    os.makedirs(OBJ, exist_ok=True)
    with open(key, "w") as f:
        f.write(built_for)
    return BIND


def build(verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(_compile, srcs))
    if os.path.exists(LIB) and os.path.getmtime(LIB) >= max(os.path.getmtime(o) for o in objs):
        build_binding()
        return LIB
    _, libdir = nccl_dirs()
    cmd = [NVCC] + ARCH + ["-shared", "-o", LIB] + objs + [
        "-L", libdir, "-l:libnccl.so.2", "-Xlinker", "-rpath," + libdir, "-cudart", "static"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    bound = build_binding()
    if verbose:
        print("built", LIB)
        if bound is None:
            print("no CUDA torch: rustgears_b200.serving has no binding")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
