"""Builds the native library in-tree.

  cutt_b200/lib/libcutt.so          shared library (C++ API + C ABI), CUDA runtime linked statically
  cutt_b200/lib/libcutt.a           static archive, the drop-in for the original libcutt.a
                                    (consumers link it with g++ ... -lcutt -lcudart)
  cutt_b200/lib/libcutt_hostcheck.so  test-only: planner + host-side plan interpreter (no CUDA)

Device code is compiled for sm_100a only.
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
OBJDIR = os.path.join(HERE, "build")

NVCC = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
GENCODE = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xptxas", "-v"] + GENCODE
CXX_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-Wall", "-Wno-unknown-pragmas"]

CU_SOURCES = ["kernels.cu", "bulk_copy.cu", "small_elt.cu", "tma_transpose.cu", "tile2d.cu", "cutt.cu",
              "rows_map.cu", "rows_move.cu", "pages.cu", "rows_api.cu"]
CXX_SOURCES = ["planner.cpp", "rows_plan.cpp"]
HEADERS = ["permute_desc.h", "permute_tile_impl.h", "planner.h", "kernels.h", "cost_model_data.h", "rowcopy_impl.h", "small_elt_impl.h",
           "tma_transpose.h", "tile2d.h",
           os.path.join("..", "..", "include", "cutt.h"), os.path.join("..", "..", "include", "cutt_c.h"),
           os.path.join("..", "..", "include", "cutt_mg.h")]
# row operators: their headers, and the sources that include them
ROWS_HEADERS = ["rows.h", "rows_plan.h", os.path.join("..", "..", "include", "cutt_rows.h")]
ROWS_SOURCES = ["rows_map.cu", "rows_move.cu", "pages.cu", "rows_api.cu", "rows_plan.cpp", "cutt.cu"]


def _newer(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def _run(cmd, log=None):
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if log is not None:
        log.write("$ " + " ".join(cmd) + "\n" + res.stdout + "\n")
    if res.returncode != 0:
        sys.stderr.write(res.stdout)
        raise RuntimeError("build step failed: " + " ".join(cmd))
    return res.stdout


def build(force: bool = False, verbose: bool = False) -> dict:
    os.makedirs(LIBDIR, exist_ok=True)
    os.makedirs(OBJDIR, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.abspath(__file__)]
    rows_hdrs = [os.path.join(CSRC, h) for h in ROWS_HEADERS]
    objs = []

    def deps(src):
        return hdrs + (rows_hdrs if src in ROWS_SOURCES else [])
    with open(os.path.join(OBJDIR, "build.log"), "a") as log:
        todo = []
        for src in CU_SOURCES + CXX_SOURCES:
            s = os.path.join(CSRC, src)
            o = os.path.join(OBJDIR, src + ".o")
            if force or _newer(o, [s] + deps(src)):
                tool = [NVCC] + NVCC_FLAGS if src in CU_SOURCES else ["g++"] + CXX_FLAGS
                todo.append(tool + ["-c", s, "-o", o])
            objs.append(o)
        # the sources do not depend on one another: half a minute to two for some of them
        with concurrent.futures.ThreadPoolExecutor(os.cpu_count() or 1) as pool:
            for out in pool.map(lambda cmd: _run(cmd, log), todo):
                if verbose:
                    print(out)
        so = os.path.join(LIBDIR, "libcutt.so")
        if force or _newer(so, objs):
            _run([NVCC, "-shared", "-o", so] + objs + GENCODE, log)
        ar = os.path.join(LIBDIR, "libcutt.a")
        if force or _newer(ar, objs):
            if os.path.exists(ar):
                os.remove(ar)
            _run(["ar", "rcs", ar] + objs, log)
        hc = os.path.join(LIBDIR, "libcutt_hostcheck.so")
        hsrc = [os.path.join(CSRC, "host_interp.cpp"), os.path.join(CSRC, "planner.cpp"), os.path.join(CSRC, "host_rows.cpp"),
                os.path.join(CSRC, "rows_plan.cpp")]
        if force or _newer(hc, hsrc + hdrs + rows_hdrs):
            _run(["g++"] + CXX_FLAGS + ["-shared", "-o", hc] + hsrc, log)
    return {"so": so, "a": ar, "hostcheck": hc}


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
