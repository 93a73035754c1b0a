"""The host stand-in of libamem_nccl (build_standin.py) with the entry points of include/amem_kv.h: their own source, over launchers
that only say that they were called. For CPU tests of what those calls refuse while the process is paused."""
import os
import subprocess

import build_standin as B


def build(outdir):
    B.build(os.path.join(B.HERE, "_build"))                  # the other objects, built where they are kept
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    lib = os.path.join(str(outdir), "libamem_nccl_kv_hoststandin.so")
    objs = [os.path.join(B.HERE, "_build", name + ".o") for name in B.PRODUCT_SOURCES + B.STANDIN_SOURCES]
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Wall", "-Wextra", "-Wno-unused-parameter", "-Wno-unused-result",
                    "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(rocm, "include"), "-shared", os.path.join(B.CSRC, "kv_api.cpp"),
                    os.path.join(B.HERE, "kv_host.cpp")] + objs + ["-o", lib, "-lpthread"], check=True, capture_output=True, text=True)
    return lib
