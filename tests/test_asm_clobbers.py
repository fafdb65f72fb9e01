"""CPU test of the kernels' inline assembly: a statement that writes m0, vcc, exec or scc names it among what it
changes, so that the compiler keeps nothing of its own there."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "nebula_amd" / "csrc"
WRITES = {
    "m0": r"\bs_\w+ m0\b", "vcc": r"\b[sv]_\w+ vcc\b", "exec": r"\bs_\w+ exec\b|_saveexec_",
    "scc": r"\bs_(?:add|sub|and|or|xor|not|cmp|lshl|lshr|ashr|bfe|min|max|abs)\w* ",
}


def statements(text):
    """(template, the clobbers' part) of each asm statement."""
    for m in re.finditer(r"\basm\s+volatile\s*\(", text):
        depth, i, quoted, parts = 1, m.end(), False, [""]
        while depth:
            ch = text[i]
            if ch == '"' and text[i - 1] != "\\":
                quoted = not quoted
            if not quoted and ch == "(":
                depth += 1
            if not quoted and ch == ")":
                depth -= 1
            if not quoted and ch == ":" and depth == 1:
                parts.append("")
            elif depth:
                parts[-1] += ch
            i += 1
        yield parts[0], parts[3] if len(parts) > 3 else ""


@pytest.mark.parametrize("source", sorted(p.name for p in CSRC.glob("*.hip")) + sorted(p.name for p in CSRC.glob("*.hpp")))
def test_registers_that_asm_writes_are_named(source):
    text = re.sub(r"//[^\n]*", "", (CSRC / source).read_text())
    for template, clobbers in statements(text):
        for register, pattern in WRITES.items():
            if re.search(pattern, template):
                assert f'"{register}"' in clobbers, f"{source}: {' '.join(template.split())}"


def test_the_scan_finds_them():
    (a, b), (c, d) = statements('asm volatile("s_mov_b32 m0, %0\\n" : : "s"(f(to)) : "memory", "m0"); asm volatile("" : "+v"(x));')
    assert "m0" in a and '"m0"' in b and re.search(WRITES["m0"], a) and c.strip() == '""' and d == ""
