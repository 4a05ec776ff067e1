"""Checks on the generated gfx950 code of the head in 8-bit integers (``int8_tiles.hip``, ``int8_few.hip``; no GPU needed).  The tiles' products are MFMAs in
assembly statements, whose hazards the compiler does not see: they are held to the distances of ``test_adapter_isa.py`` (a 16 x 16 x 64 product of 8-bit
integers takes the eight passes of one of 16 x 16 x 32 bf16 values).  No kernel spills; packed fp32 arithmetic appears in none."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest
from test_adapter_isa import bodies, faults

from skyrl_amd.csrc import build as B

pytestmark = pytest.mark.skipif(
    not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")), reason="hipcc not available"
)


def assembly(source, folder):
    out = folder / (source + ".s")
    flags = [f for f in B.HIPCC_FLAGS if f not in ("-shared", "-fPIC")]
    cmd = [shutil.which("hipcc") or "/opt/rocm/bin/hipcc", *flags, "-S", "--cuda-device-only", "-o", str(out), os.path.join(B.HERE, source)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-2000:]
    return out.read_text()


def test_tiles(tmp_path):
    text = assembly("int8_tiles.hip", tmp_path)
    seen = []
    for name, lines, body in bodies(text):
        seen.append(name)
        products = [ln for ln in lines if ln.startswith("v_mfma")]
        forms = [re.fullmatch(r"v_mfma_i32_16x16x64_i8 (a\[\d+:\d+\]), v\[\d+:\d+\], v\[\d+:\d+\], (a\[\d+:\d+\])", ln) for ln in products]
        assert all(m and m[1] == m[2] for m in forms), name
        assert not faults(lines), (name, faults(lines)[:4])
        assert re.search(r"\.amdhsa_private_segment_fixed_size 0\n", body) and not any(ln.startswith("scratch_") for ln in lines), name
    for expect in ("int8_fwd_tiles", "int8_fwd_half_tiles", "int8_logits_tiles", "int8_logits_half_tiles"):
        assert any(expect in n for n in seen), expect
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)


@pytest.mark.parametrize("source", ["int8_few.hip", "embedding_kernels.hip", "beam_kernels.hip"])
def test_no_kernel_spills(source, tmp_path):
    text = assembly(source, tmp_path)
    sizes = re.findall(r"\.amdhsa_private_segment_fixed_size (\d+)\n", text)
    assert len(sizes) >= 6 and set(sizes) == {"0"}
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
