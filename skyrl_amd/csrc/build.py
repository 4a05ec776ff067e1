"""Build the C-ABI shared library of the fused LM-head path for gfx950 with hipcc.

Usage: ``python -m skyrl_amd.csrc.build`` (or ``build()`` from Python).  The library is written next to the sources as
``libskyrl_lmhead.so``; nothing is installed outside the source tree.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_NAME = "libskyrl_lmhead.so"
SOURCES = ["lmhead_kernels.hip", "few_tokens.hip", "packed_kernels.hip", "loss_kernels.hip", "logits_kernels.hip",
           "top_logits_kernels.hip", "adapter_tiles.hip", "adapter_kernels.hip", "embedding_kernels.hip", "beam_kernels.hip",
           "int8_tiles.hip", "int8_few.hip"]
# -packed-fp32-ops off: the compiler must not form v_pk_{add,mul,fma}_f32 from the scalar fp32 epilogue code.
HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
    "-Wno-inline-asm",  # the copy instruction names M0 as clobbered; clang warns that M0 is a reserved register
]


NODE_NAME = "lookup_node.so"
NODE_SOURCE = "lookup_node.cpp"


def node_path() -> str:
    return os.path.join(HERE, NODE_NAME)


def node_command(out: str) -> list:
    """The host compiler's line for the autograd node, a Python extension against the torch that is installed."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    includes = [*cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"]]
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-isystem{d}" for d in includes], os.path.join(HERE, NODE_SOURCE), "-o", out,
            *[f"-L{d}" for d in cpp_extension.library_paths()], "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_python"]


def lib_path() -> str:
    return os.path.join(HERE, LIB_NAME)


def build(verbose: bool = False, extra_flags=(), out: str | None = None) -> str:
    """Compile the library and, next to it, the autograd node.  ``extra_flags`` / ``out``: a variant build (the timing-only ablations of
    ``skyrl_amd/bench_ablations.py``) of the library alone, written somewhere else than the product."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        raise RuntimeError("hipcc not found: the fused LM-head library can only be built with the ROCm toolchain")
    with_node = out is None
    out = out or lib_path()
    # The sources side by side into a temporary folder, and the library under a temporary name that is renamed, so a failed build never leaves a
    # half-written one behind.
    flags = [f for f in (*HIPCC_FLAGS, *extra_flags) if f != "-shared"]

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")

    with tempfile.TemporaryDirectory() as objects:
        targets = [os.path.join(objects, s + ".o") for s in SOURCES]
        node = os.path.join(objects, NODE_NAME)
        jobs = [[hipcc, *flags, "-c", "-o", o, os.path.join(HERE, s)] for s, o in zip(SOURCES, targets)]
        with concurrent.futures.ThreadPoolExecutor(8) as pool:
            list(pool.map(run, jobs + ([node_command(node)] if with_node else [])))
        fd, tmp = tempfile.mkstemp(suffix=".so", dir=os.path.dirname(out) or ".")
        os.close(fd)
        try:
            run([hipcc, *flags, "-shared", "-o", tmp, *targets])
        except RuntimeError:
            os.unlink(tmp)
            raise
        if with_node:
            shutil.move(node, node_path() + ".tmp")
            os.replace(node_path() + ".tmp", node_path())
    os.replace(tmp, out)
    os.chmod(out, 0o755)
    return out


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
