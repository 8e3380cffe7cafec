"""The scan of tests/test_isa_lds_waits.py over the 4-bit products' kernels, which read LDS with inline asm and wait for it apart, and
what their register use must stay below for the workgroups a CU that their tiles are chosen for."""
import re
import subprocess
from pathlib import Path

import pytest

from tests.test_isa_lds_waits import CSRC, HIPCC, REPO, lds_wait_hazards


def _assembly(source, tmp_path):
    cmd = [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-S", "--offload-device-only",
           "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
           "-I", str(REPO / "include"), "-I", str(CSRC), str(CSRC / source), "-o", str(tmp_path / "k.s")]
    res = subprocess.run(cmd, cwd=tmp_path, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    asm = (tmp_path / "k.s").read_text()
    bodies = {}
    for k in re.findall(r"^\s*\.type\s+(_Z\w+),@function", asm, re.M):
        i = asm.index(k + ":")
        bodies[k] = asm[i:asm.index(".Lfunc_end", i)]
    return asm, bodies


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not found")
def test_products(tmp_path):
    asm, bodies = _assembly("mx4_api.hip", tmp_path)
    for name in ("mx4_tile_kernel", "mx4_wide_kernel", "mx4_rows16_kernel", "mx4_rows_kernel", "mx4_quantise"):
        assert any(name in k for k in bodies), name
    report = {}
    for k, body in bodies.items():
        bad = lds_wait_hazards(body.split("\n"))
        if bad:
            report[k] = bad[:4]
        # f32 arithmetic two at a time has given wrong results on this chip
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", body), k
    assert not report, f"LDS read registers used before their wait: {report}"
    # operands that a call or an address keeps in memory would be read there before they arrive
    sizes = dict(zip(re.findall(r"\.name:\s+(_Z\w+)", asm), re.findall(r"\.private_segment_fixed_size: (\d+)", asm)))
    assert sizes and not any(int(v) for v in sizes.values()), sizes


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not found")
def test_rotary(tmp_path):
    asm, bodies = _assembly("rotary_api.hip", tmp_path)
    assert bodies and not any(re.search(r"\bv_pk_(add|mul|fma)_f32\b", b) for b in bodies.values())
    assert not any(int(v) for v in re.findall(r"\.private_segment_fixed_size: (\d+)", asm))
