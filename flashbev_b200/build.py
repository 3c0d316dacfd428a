"""Builds libfbev.so (sm_100a only) in-tree with nvcc.  No torch headers are involved.

    python -m flashbev_b200.build [--force]

The shared library is written next to this file so that it travels with the source
tree; it is the only native artefact of the package.
"""
from __future__ import annotations

import fcntl
import hashlib
import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(os.path.dirname(PKG_DIR), "include")
LIB_PATH = os.path.join(PKG_DIR, "libfbev.so")
SOURCES = ["fbev_kernels.cu", "fbev_query.cu", "fbev_hash.cu"]
HEADERS = sorted(os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith(".cuh")) + \
          [os.path.join(INCLUDE, h) for h in ("fbev.h", "fbev_debug.h", "fbev_query.h")]
OBJ_DIR = os.path.join(PKG_DIR, "build")  # object files, one per source, kept under the hash of what they depend on
HASH_PATH = LIB_PATH + ".srchash"  # hash of the sources the library beside it was built from

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def find_nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: libfbev.so cannot be built (CUDA 12.8+ with sm_100a support is required)")
    return cand


def source_hash() -> str:
    """SHA-256 over the library's sources and the compiler flags, in a fixed order."""
    h = hashlib.sha256(" ".join(NVCC_FLAGS).encode())
    for path in [os.path.join(CSRC, s) for s in SOURCES] + HEADERS:
        h.update(os.path.basename(path).encode())
        with open(path, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


def is_stale() -> bool:
    """True when the library is missing or was built from other sources than the ones present (compared by
    content, not by time stamp: a copied tree keeps its library and must not rebuild it)."""
    if not (os.path.exists(LIB_PATH) and os.path.exists(HASH_PATH)):
        return True
    with open(HASH_PATH) as fh:
        return fh.read().strip() != source_hash()


def _depends_on(path: str) -> list:
    """The source and every header of this library it includes, directly or through another one."""
    found, todo = [], [path]
    while todo:
        p = todo.pop()
        if p in found:
            continue
        found.append(p)
        with open(p) as fh:
            names = re.findall(r'^#include "([^"]+)"', fh.read(), flags=re.M)
        todo += [h for h in HEADERS if os.path.basename(h) in names]
    return sorted(found)


def _object(source: str, digest: str, force: bool):
    """Compiles one source unless its object file is there already; returns (object file, compiler report)."""
    path = os.path.join(CSRC, source)
    # the library's own hash goes into one small source only, so that the others need not be compiled again
    define = [f'-DFBEV_SOURCE_HASH="{digest}"'] if source == "fbev_hash.cu" else []
    h = hashlib.sha256(" ".join(NVCC_FLAGS + define).encode())
    for dep in _depends_on(path):
        with open(dep, "rb") as fh:
            h.update(os.path.basename(dep).encode() + fh.read())
    obj = os.path.join(OBJ_DIR, f"{os.path.splitext(source)[0]}.{h.hexdigest()[:16]}.o")
    log = obj[:-2] + ".ptxas.txt"
    if not force and os.path.exists(obj) and os.path.exists(log):
        with open(log) as fh:
            return obj, fh.read()
    for old in os.listdir(OBJ_DIR):  # objects of earlier versions of this source
        if old.startswith(os.path.splitext(source)[0] + ".") and ".tmp" not in old:
            os.remove(os.path.join(OBJ_DIR, old))
    tmp = f"{obj}.tmp{os.getpid()}.o"
    proc = subprocess.run([find_nvcc()] + NVCC_FLAGS + define + ["-I", INCLUDE, "-I", CSRC, "-c", path, "-o", tmp],
                          capture_output=True, text=True)
    if proc.returncode != 0:
        if os.path.exists(tmp):
            os.remove(tmp)
        raise RuntimeError(f"nvcc failed on {source}:\n{proc.stdout}{proc.stderr}")
    with open(log, "w") as fh:
        fh.write(proc.stderr)
    os.replace(tmp, obj)
    return obj, proc.stderr


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library if it is missing or older than its sources; returns its path."""
    if not force and not is_stale():
        return LIB_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    # one process at a time: the object files are shared, and each build removes those of earlier sources.  The lock goes
    # with the process that holds it; who waited for it usually finds the library made.
    with open(os.path.join(OBJ_DIR, "lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        if not force and not is_stale():
            return LIB_PATH
        return _build(force, verbose)


def _build(force: bool, verbose: bool) -> str:
    digest = source_hash()
    with ThreadPoolExecutor(len(SOURCES)) as pool:
        made = list(pool.map(lambda s: _object(s, digest, force), SOURCES))
    report = "".join(text for _, text in made)
    if verbose:
        sys.stderr.write(report)
    tmp = LIB_PATH + f".tmp{os.getpid()}"
    proc = subprocess.run([find_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", tmp] +
                          [obj for obj, _ in made], capture_output=True, text=True)
    if proc.returncode != 0:
        if os.path.exists(tmp):
            os.remove(tmp)
        raise RuntimeError(f"nvcc failed linking libfbev.so:\n{proc.stdout}{proc.stderr}")
    os.replace(tmp, LIB_PATH)  # atomic: a process loading the library meanwhile sees the old or the new file
    with open(HASH_PATH, "w") as fh:
        fh.write(digest + "\n")
    with open(os.path.join(PKG_DIR, "libfbev.ptxas.txt"), "w") as fh:  # register / spill report of the build
        fh.write(report)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
