"""Compiles the CUDA library in-tree with nvcc for sm_100a.

``python kapy-lang_b200/build.py`` (or ``build()`` from Python) produces
``kapy-lang_b200/libkapyb.so``; nvcc cross-compiles without a GPU.  The
translation units are compiled side by side into ``_obj/`` and only again when
one of the files they include changed.
"""
from __future__ import annotations

import os
import subprocess
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
SO_PATH = os.path.join(_HERE, "libkapyb.so")
_UNITS = ["kapyb_abi", "kapyb_rows"]  # csrc/<unit>.cu
_OBJ = os.path.join(_HERE, "_obj")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
]


def _sources():
    out = [os.path.join(_HERE, "..", "include", "kapyb.h")]
    d = os.path.join(_HERE, "csrc")
    out += [os.path.join(d, f) for f in sorted(os.listdir(d)) if f.endswith((".cu", ".cuh", ".h"))]
    return out


def is_stale() -> bool:
    if not os.path.exists(SO_PATH):
        return True
    t = os.path.getmtime(SO_PATH)
    return any(os.path.getmtime(s) > t for s in _sources() if os.path.exists(s))


def _unit_inputs(unit: str):
    """Files the unit's object was made from, as nvcc listed them; None before the first build."""
    dep = os.path.join(_OBJ, unit + ".d")
    if not os.path.exists(dep):
        return None
    with open(dep) as f:
        words = f.read().replace("\\\n", " ").split(":", 1)[-1].split()
    return [w for w in words if not w.startswith("/usr/")]


def _unit_stale(unit: str, flags) -> bool:
    obj = os.path.join(_OBJ, unit + ".o")
    cmd = os.path.join(_OBJ, unit + ".cmd")
    inputs = _unit_inputs(unit)
    if inputs is None or not os.path.exists(obj) or not os.path.exists(cmd):
        return True
    with open(cmd) as f:
        if f.read() != " ".join(flags):
            return True
    t = os.path.getmtime(obj)
    return any(not os.path.exists(i) or os.path.getmtime(i) > t for i in inputs)


def build(force: bool = False, verbose: bool = False) -> str:
    """KAPYB_DEBUG_SWITCHES=1 in the environment compiles the profiling switches
    that make kernels skip work (and the epilogue's per-phase clock probes) in."""
    if not force and not is_stale():
        return SO_PATH
    nvcc = os.environ.get("NVCC", "nvcc")
    flags = list(NVCC_FLAGS)
    if os.environ.get("KAPYB_DEBUG_SWITCHES", "") not in ("", "0"):
        flags.insert(0, "-DKAPYB_DEBUG_SWITCHES")
    os.makedirs(_OBJ, exist_ok=True)
    running = []
    for unit in _UNITS:
        if not force and not _unit_stale(unit, flags):
            continue
        stem = os.path.join(_OBJ, unit)
        cmd = [nvcc, *flags, "-c", "-MMD", "-MF", stem + ".d", "-o", stem + ".o",
               os.path.join(_HERE, "csrc", unit + ".cu")]
        if verbose:
            cmd[1:1] = ["-Xptxas", "-v"]
            print(" ".join(cmd), file=sys.stderr)
        if os.path.exists(stem + ".cmd"):
            os.remove(stem + ".cmd")
        running.append((unit, cmd, subprocess.Popen(cmd)))
    failed = [(cmd, p.returncode) for _, cmd, p in running if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(failed[0][1], failed[0][0])
    for unit, _, _ in running:
        with open(os.path.join(_OBJ, unit + ".cmd"), "w") as f:
            f.write(" ".join(flags))
    link = [nvcc, *NVCC_FLAGS, "-shared", "-o", SO_PATH] + [os.path.join(_OBJ, u + ".o") for u in _UNITS]
    subprocess.run(link, check=True)
    return SO_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(SO_PATH)
