"""Builds the emulated library as a shared object (TEST INFRASTRUCTURE).

The same sources and emulated device as build_emu.py, with AddressSanitizer, as
tests/emu/_build/lib/libsquirrel_emu.so: sqhip loads it where SQHIP_LIB names
it, so tests of the Python entry points run against the kernels on the CPU.
The process needs the sanitizer's runtime preloaded (`preload()`).

    python tests/emu/build_emu_lib.py
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import build_emu  # noqa: E402

OUT = os.path.join(build_emu.BUILD, "lib")
LIB = os.path.join(OUT, "libsquirrel_emu.so")
FLAGS = ["-O1", "-g", "-fno-omit-frame-pointer", "-ffp-contract=off", "-fPIC", "-fsanitize=address", "-shared-libsan"]


def preload() -> str:
    """The sanitizer's runtime, for LD_PRELOAD."""
    found = glob.glob("/opt/rocm*/lib/llvm/lib/clang/*/lib/*/libclang_rt.asan*.so")
    found = [f for f in found if "x86_64" in f]
    if not found:
        raise RuntimeError("no AddressSanitizer runtime next to the compiler")
    return sorted(found)[0]


def _compile(src: str):
    obj = os.path.join(OUT, os.path.basename(src) + ".o")
    headers = [os.path.join(build_emu.CSRC, h) for h in os.listdir(build_emu.CSRC) if h.endswith(".h")]
    headers += [os.path.join(HERE, "include", "hip", "hip_runtime.h"),
                os.path.join(build_emu.REPO, "include", "squirrel_hip.h"), __file__]
    if os.path.exists(obj) and os.path.getmtime(obj) > max(map(os.path.getmtime, [src, *headers])):
        return obj, "", 0
    tmp = f"{obj}.{os.getpid()}.tmp"
    cmd = [build_emu.CLANG, "-std=c++17", *FLAGS, "-D__HIPCC__", "-I", os.path.join(HERE, "include"), "-I",
           build_emu.CSRC, "-Wno-unused-command-line-argument", "-c", src, "-o", tmp]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode == 0:
        os.replace(tmp, obj)
    return obj, p.stdout + p.stderr, p.returncode


def build() -> str:
    os.makedirs(OUT, exist_ok=True)
    srcs = [s for s in build_emu.sources(True) if os.path.basename(s) not in ("emu_model.cpp", "selftest.cpp")]
    objs = []
    with cf.ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as ex:
        for obj, out, rc in ex.map(_compile, srcs):
            if rc:
                print(out, file=sys.stderr)
                raise RuntimeError(f"compile failed: {obj}")
            objs.append(obj)
    tmp = f"{LIB}.{os.getpid()}.tmp"
    p = subprocess.run([build_emu.CLANG, *FLAGS, "-shared", *objs, "-o", tmp, "-lm", "-lpthread"],
                       capture_output=True, text=True)
    if p.returncode:
        print(p.stdout + p.stderr, file=sys.stderr)
        raise RuntimeError("link failed")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build())
