"""Builds libesm_b200.so in-tree (esm-cpp_b200/esm_b200/libesm_b200.so).

Device translation units (csrc/*.cu) are compiled by nvcc for sm_100a only
(-gencode arch=compute_100a,code=sm_100a); the C++ host (csrc/host/*.cpp) by
g++ with the reference's release flags (-O3 -fno-math-errno), so host-side
float code such as the RoPE tables rounds exactly like the reference's.
The CUDA runtime is linked statically: the library needs only the driver.

The Python binding of the serving operators (csrc/binding/serving_ext.cpp,
against torch's headers) becomes esm_b200/_serving_ext<suffix>.so beside it.
The library does not depend on it: without torch, or with one built without
CUDA, the binding is left out, and where it fails to build that is raised when
the library is done.

    python esm-cpp_b200/build.py [--force] [--jobs N]
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.metadata
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent
REPO = PKG_ROOT.parent
CSRC = PKG_ROOT / "csrc"
OUT_SO = PKG_ROOT / "esm_b200" / "libesm_b200.so"
OBJ = PKG_ROOT / "_build"
EXT_SRC = CSRC / "binding" / "serving_ext.cpp"
OUT_EXT = PKG_ROOT / "esm_b200" / ("_serving_ext" + sysconfig.get_config_var("EXT_SUFFIX"))
EXT_TORCH = OBJ / "serving_ext.torch"  # the torch that the binding was built against

CUDA_HOME = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
NVCC = str(CUDA_HOME / "bin" / "nvcc")
GENCODE = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = GENCODE + [
    "-O3", "-std=c++17", "-lineinfo", "--fmad=false", "-Xcompiler", "-fPIC",
    "-Xptxas", "-warn-spills", f"-I{CSRC}", f"-I{REPO / 'include'}",
]
CXX = shutil.which("g++") or "g++"
CXX_FLAGS = [
    "-O3", "-fno-math-errno", "-std=c++20", "-fPIC", "-Wall", "-Wno-unused-function",
    f"-I{CSRC}", f"-I{CSRC / 'host'}", f"-I{REPO / 'include'}", f"-I{CUDA_HOME / 'include'}",
]


def _sources():
    cu = sorted(CSRC.glob("*.cu"))
    cpp = sorted((CSRC / "host").glob("*.cpp"))
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted((CSRC / "host").glob("*.h")) + [REPO / "include" / "esm_b200.h"]
    return cu, cpp, headers


def _compile(src: Path, force: bool, newest_header: float) -> Path:
    obj = OBJ / (src.stem + (".cu.o" if src.suffix == ".cu" else ".o"))
    if not force and obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, newest_header):
        return obj
    if src.suffix == ".cu":
        cmd = [NVCC, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    else:
        cmd = [CXX, *CXX_FLAGS, "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


def _torch_version() -> str:
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return ""


def binding_torch():
    """torch, if the binding can be built against it, else why not."""
    try:
        import torch
    except ModuleNotFoundError:
        return None, "torch is not installed"
    if torch.version.cuda is None:
        return None, "torch was built without CUDA"
    return torch, ""


def _build_ext(force: bool) -> None:
    header = REPO / "include" / "esm_b200.h"
    version = _torch_version()
    if (not force and OUT_EXT.exists() and EXT_TORCH.exists() and EXT_TORCH.read_text() == version
            and OUT_EXT.stat().st_mtime >= max(EXT_SRC.stat().st_mtime, header.stat().st_mtime)):
        return
    torch, why = binding_torch()
    if torch is None:
        print(f"{why}: the library is built without the serving operators' Python binding")
        return
    from torch.utils.cpp_extension import include_paths, library_paths

    cmd = [CXX, "-O2", "-std=c++20", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_serving_ext",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{REPO / 'include'}",
           f"-I{CUDA_HOME / 'include'}", f"-I{sysconfig.get_paths()['include']}",
           *(f"-I{p}" for p in include_paths()), str(EXT_SRC), "-o", str(OUT_EXT),
           *(f"-L{p}" for p in library_paths()), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    EXT_TORCH.write_text(version)


def build(force: bool = False, jobs: int | None = None, verbose: bool = True) -> Path:
    """Compiles and links the library; returns the path of the .so."""
    OBJ.mkdir(exist_ok=True)
    cu, cpp, headers = _sources()
    newest_header = max(h.stat().st_mtime for h in headers)
    srcs = cu + cpp
    with cf.ThreadPoolExecutor(max_workers=jobs or min(8, len(srcs))) as ex:
        ext = ex.submit(_build_ext, force)
        objs = list(ex.map(lambda s: _compile(s, force, newest_header), srcs))
    newest_obj = max(o.stat().st_mtime for o in objs)
    if force or not OUT_SO.exists() or OUT_SO.stat().st_mtime < newest_obj:
        cmd = [CXX, "-shared", "-o", str(OUT_SO), *map(str, objs),
               f"-L{CUDA_HOME / 'lib64'}", "-lcudart_static", "-lrt", "-ldl", "-lpthread"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    ext.result()  # raises what stopped the binding
    if verbose:
        print(f"built {OUT_SO.relative_to(REPO)}")
    return OUT_SO


def main(argv=None) -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    a = ap.parse_args(argv)
    build(force=a.force, jobs=a.jobs)
    return 0


if __name__ == "__main__":
    sys.exit(main())
