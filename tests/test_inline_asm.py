"""Inline assembly of the kernels' sources: a register that a statement names as its
instructions' destination outside its operands is declared as overwritten."""
import glob
import os
import re

from conftest import ROOT

CSRC = os.path.join(ROOT, "ml-edsl_amd", "csrc")


def statements():
    for path in sorted(glob.glob(os.path.join(CSRC, "*"))):
        text = open(path).read() if os.path.isfile(path) else ""
        for m in re.finditer(r"\basm\s*(?:volatile)?\s*\((.*?)\);", text, flags=re.S):
            if ":" in m.group(1):
                yield os.path.basename(path), m.group(1)


def test_written_registers_are_declared():
    seen = 0
    for path, body in statements():
        code, clobbers = body.split(":", 1)[0], body.rsplit(":", 1)[1]
        for line in re.split(r"\\n|\n", code):
            m = re.match(r'[\s"\\t]*\w+\s+(m0|exec|vcc|[sv]\d+|[sv]\[\d+:\d+\])\b', line)
            if m:
                seen += 1
                assert f'"{m.group(1)}"' in clobbers, (path, line)
    assert seen >= 1  # the load to LDS
