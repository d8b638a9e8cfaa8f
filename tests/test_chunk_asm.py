"""The loads to LDS that the kernels of long conversations write in assembly, against what the compiler makes around them (no GPU)."""

from __future__ import annotations

import subprocess

import pytest

from klcquant_amd import _build
from test_attention_asm import outside_and_inside


@pytest.mark.parametrize("name", ["klc_chunk.hip", "klc_key_weights.hip"])
def test_nothing_but_the_lds_loads_uses_m0(name):
    try:
        cc = _build.hipcc()
    except RuntimeError:
        pytest.skip("hipcc is not installed")
    cmd = [cc, *_build.HIPCC_FLAGS, "--cuda-device-only", "-S", str(_build.CSRC / name), "-o", "-"]
    proc = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0, proc.stderr[-2000:]
    outside, inside = outside_and_inside(proc.stdout)
    assert outside == [] and inside > 50, (inside, outside[:5])
