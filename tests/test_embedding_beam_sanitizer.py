"""The host side of the embedding and of beam search under UndefinedBehaviorSanitizer (host code only; the device code is compiled as usual): workspace
queries and argument checks over sizes at and beyond the 32- and 64-bit limits, in a child process that undefined behaviour kills."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import textwrap

import pytest

from skyrl_amd.csrc import build as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.skipif(
    not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")), reason="hipcc not available"
)

DRIVER = textwrap.dedent("""
    import ctypes, itertools, sys
    sys.path.insert(0, sys.argv[2])
    from skyrl_amd import _lib
    lib = ctypes.CDLL(sys.argv[1])
    for name, (res, args) in _lib.SIGNATURES.items():
        if "embedding" in name or "beam" in name:
            f = getattr(lib, name); f.restype = res; f.argtypes = args
    p, sizes = 0x10000, (-1, 0, 1, 63, 4097, 1 << 20, 1 << 24, (1 << 24) + 1, (1 << 31) - 1, 1 << 31, 1 << 40, (1 << 63) - 1, -(1 << 63))
    for T, H, V in itertools.product(sizes, sizes, sizes):
        assert lib.skyrl_lmhead_embedding_bwd_workspace_bytes(T, H, V) >= 0
        assert lib.skyrl_lmhead_embedding_fwd(p, 0, H, p, T, H, V, float("nan"), p, None) < 0
        assert lib.skyrl_lmhead_embedding_bwd(p, 1, H, p, -1, T, H, V, 1.0, 0, p, p, 16, None) < 0
    for N, B, V, k in itertools.product(sizes, sizes, sizes, (0, 1, 128, 129, 1 << 40, -(1 << 63))):
        lib.skyrl_logits_beam_select_workspace_bytes(N, B, V, k)
        assert lib.skyrl_logits_beam_select(p, 0, V, V, p, N, B, V, k, 1.0, p, p, p, p, 0, None) < 0
    one = (ctypes.c_void_p * 1)(p)
    for a, b, c, d in itertools.product(sizes, repeat=4):
        assert lib.skyrl_logits_beam_reorder(one, one, 1, 64, 16, 64, 32, a, b, p, c, d, d, None) < 0
        assert lib.skyrl_logits_beam_reorder(one, one, a, b, c, d, 16, 1, 16, p + 4, 1, 2, 2, None) < 0
    print("done")
""")


def test_undefined_behaviour(tmp_path, monkeypatch):
    out = str(tmp_path / "sanitized.so")
    monkeypatch.setattr(B, "SOURCES", ["embedding_kernels.hip", "beam_kernels.hip"])
    B.build(extra_flags=["-Xarch_host", "-fsanitize=undefined", "-Xarch_host", "-fsanitize-trap=undefined"], out=out)
    r = subprocess.run([sys.executable, "-c", DRIVER, out, ROOT], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "done" in r.stdout, (r.returncode, r.stderr[-2000:])
