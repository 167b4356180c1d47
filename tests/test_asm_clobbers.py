"""Inline assembly that writes a register by name says so, else the compiler may keep a value of its own there (no GPU
needed)."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "versenext_amd", "csrc")
ASM = re.compile(r'\basm\s*(?:volatile)?\s*\(((?:"(?:[^"\\]|\\.)*"|[^";])*)\)\s*;', re.S)


def statements():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        for m in ASM.finditer(open(path).read()):
            yield os.path.basename(path), m.group(1)


@pytest.mark.parametrize("reg", ["m0", "vcc", "exec", "scc"])
def test_named_registers_are_clobbers(reg):
    """The first operand of an instruction is what it writes."""
    for name, text in statements():
        code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', text.split(":")[0]))
        written = [i.split(",")[0].split()[-1] for i in code.split("\\n\\t") if len(i.split()) > 1]
        if reg in written:
            assert f'"{reg}"' in ":".join(text.split(":")[1:]), (name, code)


def test_there_are_some():
    assert sum("s_mov_b32 m0" in text for _, text in statements()) == 2
