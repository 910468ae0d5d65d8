"""The inline assembly of tg_prompt.hip (its direct-to-LDS copies), checked in
the generated code as tests/test_asm_hazards.py does for the other sources:
no copy reads an SGPR that a VALU instruction has just written."""

import shutil
import subprocess
from pathlib import Path

import pytest

from tests.test_asm_hazards import scan, scan_inflight
from tinygiant_amd import build as B


def test_copies_are_padded(tmp_path):
    if not shutil.which(B.HIPCC) and not Path(B.HIPCC).exists():
        pytest.skip("hipcc not installed")
    out = tmp_path / "tg_prompt.s"
    flags = [f for f in B.HIP_FLAGS if f != "-fPIC"]
    src = "tg_prompt.hip"
    cmd = [B.HIPCC, *flags, *B.HIP_EXTRA.get(src, []), "--cuda-device-only", "-S", "-I", str(B.CSRC), str(B.CSRC / src),
           "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    text = out.read_text()
    assert "lds" in text
    assert scan(text) == [] and scan_inflight(text) == []
    # M0 is the copies' alone: nothing else of these kernels writes it
    writes = [ln for ln in text.splitlines() if ln.strip().startswith(("s_mov_b32 m0", "s_movk_i32 m0", "s_add_u32 m0"))]
    inside, n = False, 0
    for ln in text.splitlines():
        t = ln.strip()
        inside = True if t == ";;#ASMSTART" else False if t == ";;#ASMEND" else inside
        n += inside and t.startswith("s_mov_b32 m0")
    assert len(writes) == n
