"""Build libllattn.so (sm_100a) in-tree with nvcc, and _torch_ops.so, the eager path
of lm_ops.py over it (torch's C++ headers, the host compiler).

    python build.py            # incremental: rebuilds objects whose sources changed
    python build.py --clean    # drop objects first

Objects go to csrc/_build/, the library to the package directory, next to
the Python code that loads it. Flags: -gencode arch=compute_100a,code=sm_100a
-lineinfo -O3; LLATTN_CHECK_BOUNDS=1 in the environment adds the device-side
bounds checks of the tensor-core kernels (error word instead of a trap).
"""

from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

CSRC = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(CSRC)
ROOT = os.path.dirname(PKG)
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(CSRC, "_build")
LIB = os.path.join(PKG, "libllattn.so")
TORCH_OPS = os.path.join(PKG, "_torch_ops.so")
SOURCES = ["api.cu", "pool.cu", "latent.cu", "local_simt.cu", "gate.cu", "local_sm100.cu", "decode.cu", "profile.cu",
           "xent.cu", "orth.cu", "gated.cu", "gated_few.cu", "embed.cu", "clip.cu"]
NVCC = os.environ.get("NVCC", shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc")


def flags() -> list[str]:
    f = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
         "-I" + INCLUDE, "-I" + CSRC]
    if os.environ.get("LLATTN_CHECK_BOUNDS") == "1":
        f.append("-DLLATTN_CHECK_BOUNDS=1")
    if os.environ.get("LLATTN_TRACE", "0") not in ("", "0"):
        # diagnostic builds: 1 = forward, 2 = dK/dV, 3 = gate backward phase timestamps
        f.append("-DLLATTN_TRACE=" + os.environ["LLATTN_TRACE"])
    if os.environ.get("LLATTN_PTXAS_V") == "1":
        f += ["-Xptxas", "-v"]
    return f


def _digest(src: str, fl: list[str]) -> str:
    h = hashlib.sha256(" ".join(fl).encode())
    for name in sorted(os.listdir(CSRC)) + sorted(os.listdir(INCLUDE)):
        if name.endswith((".cuh", ".h")):
            path = os.path.join(CSRC if name.endswith(".cuh") else INCLUDE, name)
            with open(path, "rb") as fh:
                h.update(fh.read())
    with open(src, "rb") as fh:
        h.update(fh.read())
    return h.hexdigest()[:16]


def _compile(name: str, fl: list[str]) -> str:
    src = os.path.join(CSRC, name)
    obj = os.path.join(BUILD, name.replace(".cu", f".{_digest(src, fl)}.o"))
    if not os.path.exists(obj):
        cmd = [NVCC, *fl, "-c", src, "-o", obj + ".tmp"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {name}:\n{r.stdout}\n{r.stderr}")
        if r.stderr.strip() and os.environ.get("LLATTN_PTXAS_V") == "1":
            sys.stderr.write(r.stderr)
        os.replace(obj + ".tmp", obj)
        stem = name.replace(".cu", ".")
        for old in os.listdir(BUILD):  # drop objects of earlier versions of this source
            if old.startswith(stem) and old.endswith(".o") and os.path.join(BUILD, old) != obj:
                os.remove(os.path.join(BUILD, old))
    return obj


def build_torch_ops() -> None:
    """_torch_ops.so, where its source, the header or torch changed."""
    import sysconfig

    import torch

    src, home = os.path.join(CSRC, "torch_ops.cpp"), os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(NVCC))), "include")
    # g++ of the path, as nvcc takes it, whatever CXX says: a newer one may link its libstdc++ in beside
    # torch's shared one, and the two do not mix (formatting an error message crashed)
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", src, "-I" + INCLUDE,
           "-I" + os.path.join(home, "include"), "-I" + os.path.join(home, "include", "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], "-I" + cuda, "-L" + os.path.join(home, "lib"), "-L" + PKG,
           "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10", "-l:libllattn.so",
           "-Wl,-rpath,$ORIGIN"]
    h = hashlib.sha256((" ".join(cmd) + torch.__version__ + sys.version).encode())
    for path in (src, os.path.join(INCLUDE, "llattn.h")):
        with open(path, "rb") as fh:
            h.update(fh.read())
    mark = os.path.join(BUILD, "torch_ops." + h.hexdigest()[:16])
    if os.path.exists(TORCH_OPS) and os.path.exists(mark):
        return
    r = subprocess.run([*cmd, "-o", TORCH_OPS + ".tmp"], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on torch_ops.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(TORCH_OPS + ".tmp", TORCH_OPS)
    for old in os.listdir(BUILD):
        if old.startswith("torch_ops."):
            os.remove(os.path.join(BUILD, old))
    open(mark, "w").close()


def build(clean: bool = False) -> str:
    if clean and os.path.isdir(BUILD):
        shutil.rmtree(BUILD)
    os.makedirs(BUILD, exist_ok=True)
    fl = flags()
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda n: _compile(n, fl), SOURCES))
    tmp = LIB + ".tmp"
    cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", *objs, "-o", tmp,
           "-Xcompiler", "-fPIC"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    build_torch_ops()
    return LIB


if __name__ == "__main__":
    print(build(clean="--clean" in sys.argv))
