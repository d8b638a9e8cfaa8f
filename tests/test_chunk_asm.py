"""The chunk attention kernels' own loads to LDS against what the compiler makes around them (no GPU)."""

from __future__ import annotations

import subprocess

import pytest

from klcquant_amd import _build
from test_attention_asm import outside_and_inside


def test_nothing_but_the_lds_loads_uses_m0():
    try:
        cc = _build.hipcc()
    except RuntimeError:
        pytest.skip("hipcc is not installed")
    cmd = [cc, *_build.HIPCC_FLAGS, "--cuda-device-only", "-S", str(_build.CSRC / "klc_chunk.hip"), "-o", "-"]
    proc = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0, proc.stderr[-2000:]
    outside, inside = outside_and_inside(proc.stdout)
    assert outside == [] and inside > 100, (inside, outside[:5])
