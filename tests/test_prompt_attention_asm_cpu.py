"""What the compiler has to know of prompt attention's tile loads, which are written in assembly: read from the IR it makes."""
import re
import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "sparse-offload-infer_amd"
sys.path.insert(0, str(PKG))


def device_ir(tmp_path, source):
    import build

    out = tmp_path / "ir.ll"
    subprocess.run([build._hipcc(), *build.HIPCC_FLAGS, "--cuda-device-only", "-emit-llvm", "-S", str(build.CSRC / source), "-o",
                    str(out)], check=True, capture_output=True)
    return out.read_text()


def test_tile_loads_state_what_they_write_and_wait_for(tmp_path):
    """m0 is among what the assembly changes, and its load comes 5 wait states after its first instruction: the most that a
    vector instruction's write to the descriptor's scalar registers needs, which the compiler does not count inside it (one
    for the write to m0)."""
    blocks = re.findall(r'asm sideeffect "([^"]*buffer_load[^"]*)", "([^"]*)"', device_ir(tmp_path, "prompt_attention.hip"))
    assert len(blocks) >= 12
    for text, constraints in blocks:
        assert "~{m0}" in constraints.split(","), constraints
        steps = [x.strip() for x in re.split(r"\\0A|\n", text.replace("\\09", " ")) if x.strip()]
        load = next(i for i, x in enumerate(steps) if x.startswith("buffer_load"))
        waits = [1 + int(x.split()[1]) if x.startswith("s_nop") else 1 for x in steps[:load]]
        at_m0 = next(i for i, x in enumerate(steps) if x.startswith("s_mov_b32 m0"))
        assert sum(waits) >= 5 and sum(waits[at_m0 + 1:]) >= 1, text
