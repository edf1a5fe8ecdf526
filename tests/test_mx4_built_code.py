"""What the compiler made of the 4-bit attention: properties of the gfx950 code that no run shows reliably."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "efficient_probing_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def _registers(operand):
    m = re.match(r"v\[(\d+):(\d+)\]$", operand) or re.match(r"v(\d+)$", operand)
    if not m:
        return set()
    lo, hi = int(m.group(1)), int(m.group(m.lastindex))
    return set(range(lo, hi + 1))


@pytest.mark.skipif(not (os.path.exists(HIPCC) or shutil.which("hipcc")), reason="needs hipcc")
def test_fp6_conversions_do_not_write_over_their_sources(tmp_path):
    """v_cvt_scalef32_2xpk16_fp6_f32 and its inverse write their result before they have read all of their sources."""
    out = tmp_path / "pool.s"
    subprocess.run([HIPCC if os.path.exists(HIPCC) else "hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fno-gpu-rdc",
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S", os.path.join(CSRC, "ep_mx4_pool.hip"),
                    "-o", str(out)], check=True, capture_output=True, timeout=600)
    seen = 0
    for line in out.read_text().splitlines():
        m = re.match(r"\s*(v_cvt_scalef32_2xpk16_fp6_f32|v_cvt_scalef32_pk32_f32_fp6)\s+(.*?)\s*(;.*)?$", line)
        if not m:
            continue
        seen += 1
        result, *sources = [_registers(o.strip()) for o in m.group(2).split(", ")]
        assert result and all(not result & s for s in sources), line
    assert seen > 0
