"""Checks on the generated gfx950 code of the tiles with adapters (``adapter_tiles.hip``; no GPU needed).  Their mainloops and the adapters' products
are MFMAs in assembly statements, whose hazards the compiler does not see, and the accumulators have to stay where the mainloop put them:

* no kernel uses scratch memory, but for dz on half tiles, which spills a few values of its epilogue and no accumulator;
* every MFMA accumulates in place; nothing else touches a register that an MFMA has written within 11 wait states (what an eight-pass MFMA's
  result takes), unless it is the MFMA that accumulates onto it;
* an accumulator or operand that was written by anything else is not read by an MFMA within two wait states.
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from skyrl_amd.csrc import build as B

pytestmark = pytest.mark.skipif(
    not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")), reason="hipcc not available"
)

RESULT, OPERAND = 11, 2  # wait states


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    out = tmp_path_factory.mktemp("isa") / "tiles.s"
    flags = [f for f in B.HIPCC_FLAGS if f not in ("-shared", "-fPIC")]
    cmd = [shutil.which("hipcc") or "/opt/rocm/bin/hipcc", *flags, "-S", "--cuda-device-only", "-o", str(out), os.path.join(B.HERE, "adapter_tiles.hip")]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-2000:]
    return out.read_text()


def bodies(text):
    for m in re.finditer(r"^(_Z\w+):[^\n]*\n(.*?)\.end_amdhsa_kernel", text, re.M | re.S):
        lines = [ln.split(";")[0].strip() for ln in m[2].split("\n")]
        lines = [ln for ln in lines if ln and not ln.startswith(".") and not ln.endswith(":")]
        if any(ln.startswith("v_mfma") for ln in lines):
            yield m[1], lines, m[2]


def registers(operand):
    m = re.fullmatch(r"([av])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m[1], r) for r in range(int(m[2]), int(m[3]) + 1)}
    m = re.fullmatch(r"([av])(\d+)", operand)
    return {(m[1], int(m[2]))} if m else set()


def faults(lines):
    clock, made, written, found = 0, {}, {}, []
    for ln in lines:
        op, _, rest = ln.partition(" ")
        operands = [o.strip().split(" ")[0] for o in rest.split(",")] if rest else []
        if op == "s_nop":
            clock += int(operands[0]) + 1
            continue
        clock += 1
        sets = [registers(o) for o in operands]
        if op.startswith("v_mfma"):
            out, c = sets[0], sets[3]
            if out != c:
                found.append(("not in place", ln))
            for r in sets[1] | sets[2]:
                if clock - made.get(r, -99) <= RESULT:
                    found.append(("result as operand", ln))
                if clock - written.get(r, -99) <= OPERAND:
                    found.append(("operand just written", ln))
            for r in c:
                if clock - written.get(r, -99) <= OPERAND:
                    found.append(("accumulator just written", ln))
            made.update(dict.fromkeys(out, clock))
            continue
        for r in set().union(*sets):
            if clock - made.get(r, -99) <= RESULT:
                found.append(("result not settled", ln))
        if op.startswith("v_") and not op.startswith("v_cmp") and sets:
            written.update(dict.fromkeys(sets[0], clock))
    return found


def test_hazards_are_found_where_they_are():
    mfma = "v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[16:19], v[0:3]"
    assert not faults([mfma, mfma, "s_nop 10", "v_add_f32_e32 v9, v3, v4"]) and faults([mfma, "s_nop 9", "v_add_f32_e32 v9, v3, v4"])
    assert faults(["v_mov_b32_e32 v8, 0", "s_nop 0", mfma]) and not faults(["v_mov_b32_e32 v8, 0", "s_nop 1", mfma])
    assert faults(["v_mov_b32_e32 v2, 0", mfma]) and faults([mfma.replace("v[0:3]", "v[4:7]", 1)])
    acc = "v_mfma_f32_16x16x32_bf16 a[0:3], v[8:11], v[16:19], a[0:3]"
    assert faults([acc, "v_accvgpr_read_b32 v1, a2"]) and faults(["v_accvgpr_write_b32 a1, v1", acc]) and not faults([acc, acc])


def test_tiles_with_adapters(assembly):
    seen = []
    for name, lines, text in bodies(assembly):
        seen.append(name)
        scratch = [ln for ln in lines if ln.startswith("scratch_")]
        assert not [ln for ln in scratch if re.search(r"\ba(\d|\[)", ln)], name
        m = re.search(r"\.amdhsa_private_segment_fixed_size (\d+)", text)
        assert m and (("half_dz" in name and int(m[1]) <= 64) or (int(m[1]) == 0 and not scratch)), name
        assert not faults(lines), (name, faults(lines)[:4])
    for expect in ("adapter_fwd_tiles", "adapter_fwd_half_tiles", "adapter_logits_tiles", "adapter_logits_half_tiles", "adapter_bwd_dz", "adapter_bwd_half_dz"):
        assert any(expect in n for n in seen), expect
