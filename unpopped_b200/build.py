"""Builds libunpopped_sm100.so in-tree with nvcc for sm_100a (B200 only).

    python -m unpopped_b200.build          # or: python unpopped_b200/build.py

Sources: unpopped_b200/csrc/*.cu. Output: unpopped_b200/libunpopped_sm100.so, which the snapshot carries to
the GPU box. Objects are compiled in parallel and relinked only when a source or header changed. Beside it stands
unpopped_b200/_bind.<Python's ABI>.so, the serving operators' Python calls (csrc/bind.cpp, host code against torch's
headers); it is built anew when its source, torch or Python changes, and left out where there is no torch.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libunpopped_sm100.so")
BIND = os.path.join(HERE, "_bind" + sysconfig.get_config_var("EXT_SUFFIX"))
BIND_MADE_WITH = os.path.join(OBJ, "bind.txt")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr", "-I", os.path.join(ROOT, "include"),
]


def nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the sm_100a library cannot be built")


def _headers():
    return glob.glob(os.path.join(CSRC, "*.cuh")) + [os.path.join(ROOT, "include", "up_sm100.h")]


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def revision_hash_of(data: bytes, h: int = 0xCBF29CE484222325) -> int:
    for b in data:
        h = ((h ^ b) * 0x100000001B3) & 0xFFFFFFFFFFFFFFFF
    return h


def revision_hash(path: str) -> int:
    """FNV-1a 64 over a source file's bytes: the reference's revision hash (crates/unpopped/src/revision.rs)."""
    with open(path, "rb") as f:
        return revision_hash_of(f.read())


# A serving operator's kernels are in more files than the one that its revision hash is of. That one holds a line with the
# hash of the others, so the revision changes with any of them.
OPERATOR_SOURCES = {
    "rope.cu": ("divide.cuh", "rope.cuh"),
    "kv4_append.cu": ("divide.cuh", "kv4.cuh", "rope.cuh"),
    "kv4_attention.cu": ("divide.cuh", "kv4.cuh", "kv4_attention.cuh", "kv4_prompt.cu", "kv4_split.cuh", "kv4_split_128.cu",
                         "kv4_split_large.cu", "kv4_split_small.cu"),
}


def sources_line(name: str) -> str:
    """The line of csrc/<name> that stands for the operator's other sources."""
    h = 0xCBF29CE484222325
    for other in OPERATOR_SOURCES[name]:
        with open(os.path.join(CSRC, other), "rb") as f:
            h = revision_hash_of(f.read(), h)
    return f"// FNV-1a 64 of {', '.join(OPERATOR_SOURCES[name])}: {h:016x}\n"


def write_sources_lines():
    """Brings the operators' lines up to date (python -m unpopped_b200.build --sources), after any of their files changed."""
    for name in OPERATOR_SOURCES:
        path = os.path.join(CSRC, name)
        with open(path) as f:
            text = f.read()
        new = re.sub(r"// FNV-1a 64 of .*\n", lambda m: sources_line(name), text, count=1)
        if new != text:
            with open(path, "w") as f:
                f.write(new)


def _compile(src: str, extra) -> str:
    obj = os.path.join(OBJ, os.path.basename(src) + ".o")
    if _stale(obj, [src] + _headers()):
        rev = f"-DUP_SOURCE_REVISION=0x{revision_hash(src):016x}ull"
        cmd = [nvcc()] + NVCC_FLAGS + [rev] + list(extra) + ["-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{r.stdout}\n{r.stderr}")
    return obj


def build(verbose: bool = False, extra=()) -> str:
    """Compile every csrc/*.cu for sm_100a and link the shared library; returns its path."""
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, extra), srcs))
    if _stale(LIB, objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc()] + ARCH + ["-shared", "-o", tmp] + objs + ["-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    _build_bind()
    if verbose:
        print(LIB)
    return LIB


def _bind_command() -> list | None:
    """What compiles csrc/bind.cpp, without its output; None where there is no torch to compile it against."""
    if importlib.util.find_spec("torch") is None:
        return None
    import torch

    base = os.path.dirname(torch.__file__)
    if not os.path.isdir(os.path.join(base, "include", "ATen")):
        return None
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    includes = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
                sysconfig.get_paths()["include"], cuda, os.path.join(ROOT, "include")]
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + [f"-I{d}" for d in includes] +
            [os.path.join(CSRC, "bind.cpp"), "-L" + os.path.join(base, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10",
             "-lc10_cuda", "-L" + HERE, "-l:libunpopped_sm100.so", "-Wl,-rpath,$ORIGIN"])


def _bind_made_with(cmd) -> str:
    """The text that changes with whatever the binding's binary form depends on beside its source."""
    import torch

    return "\n".join([torch.__version__, sys.version, *cmd])


def _bind_stale(cmd) -> bool:
    if _stale(BIND, [os.path.join(CSRC, "bind.cpp"), os.path.join(ROOT, "include", "up_sm100.h")]):
        return True
    if not os.path.exists(BIND_MADE_WITH):
        return True
    with open(BIND_MADE_WITH) as f:
        return f.read() != _bind_made_with(cmd)


def _build_bind():
    cmd = _bind_command()
    if cmd is None:
        print("no torch headers: the C library only, without the Python calls of the serving operators", file=sys.stderr)
        return
    if not _bind_stale(cmd):
        return
    tmp = BIND + ".tmp"
    r = subprocess.run(cmd + ["-o", tmp], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on bind.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BIND)
    with open(BIND_MADE_WITH, "w") as f:
        f.write(_bind_made_with(cmd))


def ptxas_report(src_name: str) -> str:
    """Register / spill / shared-memory report of one source (nvcc -Xptxas -v)."""
    src = os.path.join(CSRC, src_name)
    cmd = [nvcc()] + NVCC_FLAGS + ["-Xptxas", "-v", "-c", src, "-o", os.devnull]
    r = subprocess.run(cmd, capture_output=True, text=True)
    return r.stdout + r.stderr


if __name__ == "__main__":
    if len(sys.argv) > 1 and sys.argv[1] == "--ptxas":
        for name in sys.argv[2:]:
            print(ptxas_report(name))
    elif sys.argv[1:] == ["--sources"]:
        write_sources_lines()
    else:
        build(verbose=True)
