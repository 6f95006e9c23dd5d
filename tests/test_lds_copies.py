"""The copies from memory straight into LDS that are written in inline assembly."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "roost_amd" / "csrc"


def test_m0_is_written_a_wait_state_before_the_copy_that_reads_it():
    """A copy takes its LDS address from M0, and an instruction that does so needs one wait state after a scalar write of M0.
    The compiler keeps to that for its own instructions and does not look into inline assembly."""
    found = 0
    for source in sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.h")]):
        for text in re.findall(r'asm volatile\("([^"]*global_load_lds[^"]*)"', source.read_text()):
            lines = [line.strip().split()[0] for line in text.split("\\n\\t")]
            copy = next(i for i, op in enumerate(lines) if op.startswith("global_load_lds"))
            write = max(i for i, line in enumerate(text.split("\\n\\t")[:copy]) if re.match(r"s_\w+ m0,", line))
            assert "s_nop" in lines[write + 1:copy], f"{source.name}: {text}"
            found += 1
    assert found >= 1
