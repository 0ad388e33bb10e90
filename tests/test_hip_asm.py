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
def test_m0_is_put_back_and_waits_are_long_enough(name, statement):
    code = instructions(statement)
    if any(re.match(r"s_mov_b32 m0\b", x) for x in code):     # the compiler reserves m0 and takes no note of it in a list of overwritten registers
        kept = re.match(r"s_mov_b32 (%\d+), m0$", code[0])
        assert kept and code[-1] == "s_mov_b32 m0, " + kept[1], (name, statement)
        assert not any(kept[1] in re.findall(r"%\d+", x) for x in code[1:-1]), (name, statement)
    for i, x in enumerate(code):
        if not x.startswith("global_load_lds"):
            continue
        states = 0                                             # between the statement's begin, and between m0's write, and the load
        since_m0 = None
        for y in code[:i]:
            n = int(y.split()[1]) + 1 if y.startswith("s_nop") else 1
            states += n
            since_m0 = 0 if y.startswith("s_mov_b32 m0") else None if since_m0 is None else since_m0 + n
        assert since_m0 is not None and since_m0 >= 1, (name, statement)
        if not x.endswith("off"):                              # its base lies in scalar registers: five states behind a vector write
            assert states >= 5, (name, statement)
