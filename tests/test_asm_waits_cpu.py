"""Inline assembly carries its own waits: the compiler places none inside or right before it.

Read from the sources, statement by statement.  An instruction between two others is one wait state, s_nop n is n + 1.
"""
import glob
import os
import re


CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "humanoid-vision-system_amd", "csrc")


def statements():
    """(file:line, instructions, constraint of each operand) of every asm statement."""
    got = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))):
        text = open(path).read()
        for m in re.finditer(r"\basm\s+volatile\s*\(", text):
            depth, at, quoted = 1, m.end(), False
            while depth:                                            # the closing bracket outside of quotes
                c = text[at]
                if c == '"' and text[at - 1] != "\\":
                    quoted = not quoted
                elif not quoted:
                    depth += (c == "(") - (c == ")")
                at += 1
            body = text[m.end():at - 1]
            code = re.match(r'\s*((?:"(?:[^"\\]|\\.)*"\s*|#\s*\w+\s*)+)', body)
            lines = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', code.group(1)))
            operands = re.findall(r'"([^"]*)"\s*\(', body[code.end():])
            got.append((f"{os.path.basename(path)}:{text.count(chr(10), 0, m.start()) + 1}",
                        [x.strip() for x in re.split(r"\\n|\\t|;", lines) if x.strip()], operands))
    return got


def waits(instructions):
    return sum(int(x.split()[1], 0) + 1 if x.startswith("s_nop") else 1 for x in instructions)


def test_statements_are_found():
    assert sum(any("lds" in x for x in code) for _, code, _ in statements()) >= 2
    assert waits(["s_mov_b32 m0, s0", "s_nop 3"]) == 5


def test_a_load_to_lds_waits_for_m0():
    """A scalar write of M0 and a load to LDS, which reads it, need one wait state between them."""
    for where, code, _ in statements():
        for i, x in enumerate(code):
            if not re.search(r"_load_lds_|\blds\b", x):
                continue
            writes = [j for j in range(i) if re.match(r"s_\w+\s+m0\b", code[j])]
            assert writes, f"{where}: {x} without its M0"
            assert waits(code[writes[-1] + 1:i]) >= 1, f"{where}: {x} right after the write of M0"


def test_a_load_waits_for_its_scalar_address():
    """A load that takes its base from a scalar pair needs five wait states after a vector instruction (a lane read) wrote the
    pair.  The operand may come from one, right before the statement, so the statement holds all five."""
    seen = 0
    for where, code, operands in statements():
        for i, x in enumerate(code):
            if not re.match(r"(global|buffer|flat|scratch)_", x):
                continue
            base = [int(n) for n in re.findall(r"%(\d+)", x) if "s" in operands[int(n)]]
            if base:
                seen += 1
                assert waits(code[:i]) >= 5, f"{where}: {x}: {waits(code[:i])} wait states"
    assert seen
