"""The inline assembly of tg_paged.hip (its direct-to-LDS copies of queries),
checked in the generated code as tests/test_prompt_asm.py does for the dense
caches, whose helpers it shares."""

import shutil
import subprocess
from pathlib import Path

import pytest

from tests.test_asm_hazards import scan, scan_inflight
from tinygiant_amd import build as B


def test_copies_are_padded(tmp_path):
    if not shutil.which(B.HIPCC) and not Path(B.HIPCC).exists():
        pytest.skip("hipcc not installed")
    src, out = "tg_paged.hip", tmp_path / "tg_paged.s"
    flags = [f for f in B.HIP_FLAGS if f != "-fPIC"]
    r = subprocess.run([B.HIPCC, *flags, *B.HIP_EXTRA.get(src, []), "--cuda-device-only", "-S", "-I", str(B.CSRC), str(B.CSRC / src),
                        "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    text = out.read_text()
    assert "lds" in text
    assert scan(text) == [] and scan_inflight(text) == []
    assert "v_pk_fma_f32" not in text and "v_pk_mul_f32" not in text and "v_pk_add_f32" not in text
    # M0 is the copies' alone: nothing else of these kernels writes it
    writes = [ln for ln in text.splitlines() if ln.strip().startswith(("s_mov_b32 m0", "s_movk_i32 m0", "s_add_u32 m0"))]
    inside, n = False, 0
    for ln in text.splitlines():
        t = ln.strip()
        inside = True if t == ";;#ASMSTART" else False if t == ";;#ASMEND" else inside
        n += inside and t.startswith("s_mov_b32 m0")
    assert len(writes) == n
