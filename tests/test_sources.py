"""Rules that the compiler cannot check, read off the kernel sources."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "padra_b200" / "csrc"


def test_registers_of_a_tensor_memory_load_are_tied_to_its_wait():
    """tcgen05.ld and tcgen05.wait::ld are statements of their own, and a memory clobber does not order arithmetic on registers: what
    was loaded has to pass through an empty statement behind the wait before it is used."""
    waits = 0
    for path in sorted(CSRC.glob("*.cu*")):
        text = path.read_text()
        for wait in re.finditer(r'asm volatile\("tcgen05\.wait::ld', text):
            body = text[wait.end():text.index("\n}", wait.end())]
            assert re.search(r'asm volatile\("" : "\+[rf]"', body), f"{path.name}: a load's registers are not tied to its wait"
            waits += 1
    assert waits == len(re.findall(r"tcgen05\.wait::ld", "".join(p.read_text() for p in CSRC.glob("*.cu*")))) > 0
