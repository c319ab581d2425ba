"""Waits that the compiler cannot add by itself: what stands in an asm block has to carry its own."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "distributedpytorch_amd" / "csrc"


def _blocks():
    """(file, text) of every asm statement in the kernels' sources."""
    for src in sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.h")]):
        text = src.read_text()
        for at in re.finditer(r"\basm\s+volatile\s*\(", text):
            yield src.name, text[at.start():text.index(");", at.end())]


def test_a_write_of_m0_is_one_wait_state_old_before_a_load_to_lds_reads_it():
    """gfx9: SALU write of M0, then a buffer load with LDS = 1: one wait state between them, and M0 named as overwritten."""
    found = 0
    for name, block in _blocks():
        code = "".join(re.findall(r'"([^"]*)"', block)).replace("\\t", "").split("\\n")
        writes = [i for i, line in enumerate(code) if re.match(r"s_mov_b32 m0\b", line)]
        loads = [i for i, line in enumerate(code) if re.match(r"buffer_load\w* .*\blds\b", line)]
        if not writes and not loads:
            continue
        found += 1
        for load in loads:
            last = max(i for i in writes if i < load)
            assert any(re.match(r"s_nop \d", line) for line in code[last + 1:load]), f"{name}: {block}"
        assert '"m0"' in block.split(":")[-1], f"{name}: {block}"
    assert found
