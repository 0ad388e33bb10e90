"""Inline assembly in the HIP sources: what the compiler cannot see has to be said (CPU-safe: the sources are read)."""
import glob
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCES = sorted(glob.glob(os.path.join(ROOT, "vectordb_amd", "csrc", "*.hip")) + glob.glob(os.path.join(ROOT, "vectordb_amd", "csrc", "*.hpp")))


def statements():
    """(file, text) of every asm statement."""
    for path in SOURCES:
        text = open(path).read()
        for m in re.finditer(r"\basm\s+volatile\s*\(", text):
            depth, quoted, i = 1, False, m.end()
            while depth:
                c = text[i]
                if c == '"' and text[i - 1] != "\\":
                    quoted = not quoted
                elif not quoted:
                    depth += (c == "(") - (c == ")")
                i += 1
            yield os.path.basename(path), text[m.end():i - 1]


def instructions(statement):
    code = " ".join(re.findall(r'"((?:[^"\\]|\\.)*)"', statement.split(":")[0])).replace("\\n", "\n").replace("\\t", " ")
    return [x.strip() for x in code.split("\n") if x.strip()]


def test_there_are_statements_to_look_at():
    assert sum("global_load_lds" in s for _, s in statements()) >= 3


@pytest.mark.parametrize("name,statement", list(statements()))
def test_m0_is_an_operand_and_waits_are_long_enough(name, statement):
    """The compiler reserves m0: it takes no note of m0 among overwritten registers, but it knows what it puts there as an operand."""
    code = instructions(statement)
    assert not any(re.match(r"s_\w+ m0\b", x) for x in code), (name, statement)
    for i, x in enumerate(code):
        if not x.startswith("global_load_lds"):
            continue
        assert '"{m0}"' in statement, (name, statement)
        states = sum(int(y.split()[1]) + 1 if y.startswith("s_nop") else 1 for y in code[:i])
        # one state behind m0's write; five where the base lies in scalar registers, which a vector instruction may have written last
        assert states >= (1 if x.endswith("off") else 5), (name, statement)
