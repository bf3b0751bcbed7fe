"""Builds libhmw4a16.so (the gfx950 kernels and the C ABI of include/hm_w4a16.h) in-tree with hipcc.

Usage: python heteromega_amd/build.py [--verbose]
"""

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD_DIR = os.path.join(HERE, "_build")
LIB_NAME = "libhmw4a16.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)

SOURCES = ["hm_api.cpp", "hm_split.cpp", "hm_layout.hip", "hm_gemv.hip", "hm_gemm.hip", "hm_gemm_f16.hip", "hm_gemm_bf16.hip", "hm_elementwise.hip", "hm_static.hip", "hm_pages.hip",
           "hm_rope.hip", "hm_paged_attention.hip", "hm_paged_attention_f16.hip", "hm_paged_attention_bf16.hip", "hm_attention_api.cpp", "hm_page_fork.hip",
           "hm_beam.hip", "hm_share_plan.hip", "hm_shared_attention.hip", "hm_shared_attention_f16.hip", "hm_shared_attention_bf16.hip", "hm_branch_api.cpp"]
ARCH = "gfx950"

COMMON_FLAGS = [
    "-O3",
    "-std=c++17",
    "-fPIC",
    f"--offload-arch={ARCH}",
    # Packed fp32 instructions are kept out of the generated code: some of their forms have given wrong results on
    # these parts without an error, so the compiler may not form them from scalar or float2 code.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-mcode-object-version=5",
    "-Wall",
    "-Wno-unused-function",
    f"-I{os.path.join(ROOT, 'include')}",
]


def hipcc():
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: the HIP extension cannot be built")


def _compile(src, verbose):
    obj = os.path.join(BUILD_DIR, os.path.splitext(src)[0] + ".o")
    lang = ["-x", "hip"] if src.endswith(".hip") else []
    cmd = [hipcc(), *lang, *COMMON_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{res.stdout}\n{res.stderr}")
    noise = [ln for ln in res.stderr.splitlines() if "packed-fp32-ops" not in ln and ln.strip()]
    if verbose and noise:
        print("\n".join(noise), flush=True)
    return obj


SHIM_DIR = os.path.join(HERE, "shim")
SHIM_SOURCES = ["hm_reference_api.cpp", "py_module.cpp"]
SHIM_NAME = "_reference_shim"
HOST_SOURCES = ["hm_attention_host.cpp", "hm_branch_host.cpp"]
HOST_NAME = "_attention_host"


def _build_extension(name, directory, sources, libs, verbose):
    """A Python module of host code (g++) against torch's C++ headers, next to the package's own."""
    import sysconfig

    import torch
    import torch.utils.cpp_extension as ext

    torch_lib = ext.library_paths()[0]
    out = os.path.join(HERE, name + sysconfig.get_config_var("EXT_SUFFIX"))
    flags = ["-O2", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             f"-DTORCH_EXTENSION_NAME={name}", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{sysconfig.get_paths()['include']}",
             *[f"-I{p}" for p in ext.include_paths()], f"-I{os.path.join(ROOT, 'include')}"]
    os.makedirs(BUILD_DIR, exist_ok=True)

    def compile_one(src):
        obj = os.path.join(BUILD_DIR, os.path.splitext(src)[0] + ".o")
        cmd = ["g++", *flags, "-c", os.path.join(directory, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"build of {name} failed on {src}:\n{res.stdout}\n{res.stderr}")
        return obj

    with ThreadPoolExecutor(max_workers=len(sources)) as pool:
        objs = list(pool.map(compile_one, sources))
    cmd = ["g++", "-shared", *objs, f"-L{torch_lib}", "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python", f"-L{HERE}", *libs,
           "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{torch_lib}", "-Wl,-rpath,$ORIGIN", "-o", out + ".tmp"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link of {name} failed:\n{res.stdout}\n{res.stderr}")
    os.replace(out + ".tmp", out)
    return out


def build_shim(verbose=False):
    """The reference-signature C++ operators (shim/hm_reference_api.cpp) against torch's C++ headers, as a Python
    module over libhmw4a16.so. Host code only (g++): it calls the C ABI and launches nothing itself."""
    return _build_extension(SHIM_NAME, SHIM_DIR, SHIM_SOURCES, ["-lhmw4a16"], verbose)


def build_host(verbose=False):
    """The compiled host side of the attention operators' Python calls (csrc/hm_attention_host.cpp)."""
    return _build_extension(HOST_NAME, CSRC, HOST_SOURCES, [], verbose)


def build(verbose=False):
    os.makedirs(BUILD_DIR, exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(len(SOURCES), 8)) as pool:
        objs = list(pool.map(lambda s: _compile(s, verbose), SOURCES))
    tmp = LIB_PATH + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    verbose = "--verbose" in sys.argv
    if "--no-shim" in sys.argv:  # the library alone, which needs none of torch's headers
        print(build(verbose))
    else:
        with ThreadPoolExecutor(max_workers=2) as pool:  # the module builds beside the library: it does not link with it
            host = pool.submit(build_host, verbose)
            print(build(verbose))
            print(host.result())
        print(build_shim(verbose))
