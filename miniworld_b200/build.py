"""Build recipe of the two in-tree libraries: the kernels behind the C ABI (``nvcc``, sm_100a only) and the native
host side of the module calls (``csrc/host.cpp``, one ``g++`` call against PyTorch's headers, linked to the first)."""

from __future__ import annotations

import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_NAME = "libb200_trimul.so"
LIB_PATH = PKG_DIR / LIB_NAME
NATIVE_PATH = PKG_DIR / "_native.so"
NATIVE_TAG_PATH = PKG_DIR / "_native.tag"  # what NATIVE_PATH was built against
HOST_SOURCE = CSRC / "host.cpp"
HEADER = PKG_DIR.parent / "include" / "b200_trimul.h"
BLOCKS_HEADER = PKG_DIR.parent / "include" / "b200_blocks.h"
BLOCKS_HOST = CSRC / "host_blocks.inc"  # part of HOST_SOURCE

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
]


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [p for p in sorted(CSRC.glob("*.inc")) if p != BLOCKS_HOST] + [HEADER, BLOCKS_HEADER]


def is_stale() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    return any(src.stat().st_mtime > built for src in _sources())


def native_tag() -> str:
    """The interpreter and the PyTorch that ``_native.so`` is bound to: with another one it does not load, or not rightly."""
    import sysconfig

    import torch

    return f"{sysconfig.get_config_var('SOABI')} torch {torch.__version__} cxx11 abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}\n"


def native_is_stale() -> bool:
    if not NATIVE_PATH.exists() or not NATIVE_TAG_PATH.exists() or NATIVE_TAG_PATH.read_text() != native_tag():
        return True
    built = NATIVE_PATH.stat().st_mtime
    return any(src.stat().st_mtime > built for src in (HOST_SOURCE, HEADER, BLOCKS_HOST, BLOCKS_HEADER, Path(__file__)))


def find_nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found: cannot build " + LIB_NAME)
    return nvcc


def _run(cmd: list[str]) -> subprocess.CompletedProcess:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed:\n" + proc.stdout + proc.stderr)
    return proc


def build_native(force: bool = False) -> Path:
    """Compile ``csrc/host.cpp`` into ``_native.so`` beside the package (needs the kernels' library to link to)."""
    if not force and not native_is_stale():
        return NATIVE_PATH
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(find_nvcc()).resolve().parent.parent
    tmp = NATIVE_PATH.with_suffix(".so.tmp")
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_native", "-DTORCH_API_INCLUDE_EXTENSION_H",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{root}/include",
          f"-I{root}/include/torch/csrc/api/include", f"-I{cuda}/include", f"-I{sysconfig.get_paths()['include']}",
          str(HOST_SOURCE), "-o", str(tmp), f"-L{root}/lib", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-ltorch_cuda", "-lc10", "-lc10_cuda",
          f"-L{PKG_DIR}", f"-l:{LIB_NAME}", "-Wl,-rpath,$ORIGIN"])
    os.replace(tmp, NATIVE_PATH)
    NATIVE_TAG_PATH.write_text(native_tag())
    return NATIVE_PATH


def _compiler_tag() -> str:
    """What an object file is made with: objects of different compilers or flags are not linked together."""
    nvcc = find_nvcc()
    return "\n".join([nvcc, *NVCC_FLAGS, _run([nvcc, "--version"]).stdout])


def _compile(source: Path, force: bool, verbose: bool) -> Path:
    """Object file of one ``.cu`` file, kept beside the package and made again when a file that it includes is newer or the compiler
    or its flags have changed."""
    obj, deps, made_with = (PKG_DIR / f"{source.stem}{end}" for end in (".o", ".tag", ".flags.tag"))
    tag = _compiler_tag()
    if not force and obj.exists() and deps.exists() and made_with.exists() and made_with.read_text() == tag:
        used = [Path(w) for w in deps.read_text().replace("\\\n", " ").split(" : ", 1)[-1].split()]
        built = obj.stat().st_mtime
        if used and all(p.exists() and p.stat().st_mtime <= built for p in used):
            return obj
    cmd = [find_nvcc(), *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-MD", "-MF", str(deps)]
    made_with.unlink(missing_ok=True)
    proc = _run(cmd + ["-c", "-o", str(obj), str(source)])
    made_with.write_text(tag)
    if verbose:
        print(proc.stderr)
    return obj


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile ``csrc/*.cu`` side by side and link them to ``libb200_trimul.so`` beside the package (no GPU needed), then
    ``_native.so``."""
    if force or is_stale():
        sources = sorted(CSRC.glob("*.cu"))
        with ThreadPoolExecutor(len(sources)) as pool:
            objects = list(pool.map(lambda source: _compile(source, force, verbose), sources))
        tmp = LIB_PATH.with_suffix(".so.tmp")
        _run([find_nvcc(), *NVCC_FLAGS, "-shared", "-o", str(tmp), *map(str, objects)])
        os.replace(tmp, LIB_PATH)
    build_native(force)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force=True, verbose=True))
