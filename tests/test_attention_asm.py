"""The attention kernels' own assembly against what the compiler makes around it (no GPU)."""

from __future__ import annotations

import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from klcquant_amd import _build

M0 = re.compile(r"(?<![\w.])m0(?!\w)")


def outside_and_inside(asm: str) -> tuple[list[str], int]:
    """The lines that name m0 outside the sources' assembly blocks, and how many do inside them."""
    own, outside, inside = False, [], 0
    for line in asm.splitlines():
        if "#ASMSTART" in line or "#ASMEND" in line:
            own = "#ASMSTART" in line
        elif M0.search(line.split(";")[0]):
            inside += own
            if not own:
                outside.append(line.strip())
    return outside, inside


def test_nothing_but_the_lds_loads_uses_m0():
    """The loads to LDS write m0, a register that the compiler reserves: it allocates nothing to it, but instructions
    that need it would be given it just before them, perhaps ahead of such a block.  So there must be none."""
    try:
        cc = _build.hipcc()
    except RuntimeError:
        pytest.skip("hipcc is not installed")

    def compiled(name):
        cmd = [cc, *_build.HIPCC_FLAGS, "--cuda-device-only", "-S", str(_build.CSRC / name), "-o", "-"]
        proc = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
        assert proc.returncode == 0, proc.stderr[-2000:]
        return proc.stdout

    names = ("klc_prompt.hip", "klc_batch.hip")
    with ThreadPoolExecutor(max_workers=2) as pool:
        for name, asm in zip(names, pool.map(compiled, names)):
            outside, inside = outside_and_inside(asm)
            assert outside == [] and inside > 100, (name, inside, outside[:5])


def test_the_check_sees_other_uses():
    asm = "\t;;#ASMSTART\n\ts_mov_b32 m0, s1\n\t;;#ASMEND\n\ts_mov_b32 m0, -1 ; comment\n\ts_add_u32 s1, s2, s3 ; m0\n"
    assert outside_and_inside(asm) == (["s_mov_b32 m0, -1 ; comment"], 1)
