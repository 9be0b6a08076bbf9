"""What the HIP sources have to keep to where the compiler cannot see to it: inside inline assembly."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "csrc" / "hip"


def _asm_blocks():
    for path in sorted(CSRC.glob("*.hip")) + sorted(CSRC.glob("*.h")):
        for m in re.finditer(r"\basm\s+volatile\s*\((.*?)\);", path.read_text(), re.S):
            lines = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', m.group(1).split(":")[0]))
            yield path.name, [s.strip() for s in re.split(r"\\n|\\t|;", lines) if s.strip()]


def test_a_write_of_m0_is_a_wait_state_ahead_of_lds_dma():
    """gfx9 asks for one wait state between a scalar write of M0 and a load into the LDS, which reads it as
    its address; the compiler puts an s_nop there, in inline assembly nobody does."""
    seen = 0
    for name, lines in _asm_blocks():
        for a, b in zip(lines, lines[1:]):
            if re.match(r"s_\w+ m0\b", a):
                assert not re.search(r"(global|buffer|scratch)_load\w*lds|_load.*\blds\b", b), (name, a, b)
        seen += any("load_lds" in s for s in lines)
    assert seen  # the pattern still finds the blocks it is about
