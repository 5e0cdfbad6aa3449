"""Build the gfx950 attention library (libsgl_attn.so) in-tree.

Each HIP source under csrc/ is compiled for gfx950 with hipcc and linked
into one shared library next to this file; the C++ backend extension
(LibTorch host code over the C ABI) is built by build_backend().
Run directly: python sglang.cpp_amd/build.py
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
BUILD_DIR = PKG_DIR / "_build"
LIB_NAME = "libsgl_attn.so"
LIB_PATH = PKG_DIR / LIB_NAME

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

# Packed-fp32 VALU ops are disabled for all device code (some packed fp32
# forms have given silently wrong results on these parts); hipcc's host pass warns that it does not know the
# feature, which is harmless.
HIP_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-fPIC",
    "-std=c++17",
    "-Wno-unused-command-line-argument",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{REPO / 'include'}",
]

SOURCES = ["kv_store.hip", "metadata.hip", "rope_norm.hip", "decode.hip", "prefill.hip", "residual.hip",
           "sampling.hip", "softmax.hip", "rope_append.hip", "verify.hip", "prefix.hip"]


def _compile(src: Path, obj: Path) -> None:
    cmd = [HIPCC, *HIP_FLAGS, "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    # Surface real diagnostics, drop the known host-pass feature warning.
    lines = [ln for ln in res.stderr.splitlines()
             if "packed-fp32-ops" not in ln and "warning: unknown" not in ln and ln.strip()]
    if lines:
        sys.stderr.write("\n".join(lines) + "\n")


def build_lib(jobs: int = 8) -> Path:
    BUILD_DIR.mkdir(exist_ok=True)
    objs = []
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        futs = []
        for name in SOURCES:
            src = CSRC / name
            obj = BUILD_DIR / (name + ".o")
            objs.append(obj)
            futs.append(ex.submit(_compile, src, obj))
        for f in futs:
            f.result()
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


BACKEND_NAME = "sgl_backend"
BACKEND_SOURCES = ["backend/hip_backend.cpp", "backend/bindings.cpp"]


def backend_path() -> Path:
    import sysconfig
    return PKG_DIR / (BACKEND_NAME + sysconfig.get_config_var("EXT_SUFFIX"))


def build_backend(jobs: int = 8) -> Path:
    """Build the C++ backend extension (host code only, LibTorch + pybind11).

    Compiled with g++ directly against torch's headers; it links
    libsgl_attn.so from this directory (rpath $ORIGIN), so all device work
    stays in the HIP library.
    """
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    cflags = [
        "-O2", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function",
        "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
        "-DTORCH_EXTENSION_NAME=" + BACKEND_NAME, "-DTORCH_API_INCLUDE_EXTENSION_H",
        f"-I{sysconfig.get_paths()['include']}", "-I/opt/rocm/include", f"-I{REPO / 'include'}",
        *[f"-I{p}" for p in cpp_extension.include_paths()],
    ]
    BUILD_DIR.mkdir(exist_ok=True)
    objs = []

    def cc(name: str) -> Path:
        src = CSRC / name
        obj = BUILD_DIR / (Path(name).stem + ".cpp.o")
        res = subprocess.run(["g++", *cflags, "-c", str(src), "-o", str(obj)],
                             capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"g++ failed for {name}:\n{res.stdout}\n{res.stderr}")
        if res.stderr.strip():
            sys.stderr.write(res.stderr)
        return obj

    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(cc, BACKEND_SOURCES))
    torch_lib = Path(torch.__file__).resolve().parent / "lib"
    out = backend_path()
    tmp = out.with_name(out.name + ".tmp")
    cmd = ["g++", "-shared", *map(str, objs), "-o", str(tmp),
           f"-L{PKG_DIR}", "-l:" + LIB_NAME, "-Wl,-rpath,$ORIGIN",
           f"-L{torch_lib}", f"-Wl,-rpath,{torch_lib}",
           "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10_hip", "-ltorch_hip",
           "-L/opt/rocm/lib", "-lamdhip64"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"backend link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, out)
    return out


PROBES_NAME = "libsgl_probes.so"
PROBES_SOURCE = "probes/ceilings.hip"


def build_probes() -> Path:
    """The hardware-ceiling probes the benchmark reports beside the
    attention kernels (stream read, MFMA issue, empty launch); a library of
    their own, outside the attention ABI."""
    BUILD_DIR.mkdir(exist_ok=True)
    obj = BUILD_DIR / "ceilings.hip.o"
    _compile(CSRC / PROBES_SOURCE, obj)
    out = PKG_DIR / PROBES_NAME
    tmp = out.with_suffix(".so.tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", str(obj), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"probe link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, out)
    return out


def build(jobs: int = 8) -> None:
    build_lib(jobs)
    build_backend(jobs)
    build_probes()


if __name__ == "__main__":
    build()
    print(LIB_PATH)
