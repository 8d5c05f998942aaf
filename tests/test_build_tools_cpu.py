"""CPU: the debug builds under tools/ compile and link what rag_amd/_build.py does: no list of flags or objects of their own."""
import glob
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("script", sorted(os.path.basename(p) for p in glob.glob(os.path.join(ROOT, "tools", "*.sh"))))
def test_compile_and_link_lines_ask_the_build(script):
    with open(os.path.join(ROOT, "tools", script)) as f:
        lines = [x for x in f if re.search(r"\bhipcc\b", x) and not x.lstrip().startswith("#")]
    for line in lines:
        want = "$(python -m rag_amd._build --objects" if "-shared" in line else "$(python -m rag_amd._build --flags"
        assert want in line, line
    assert lines or not script.startswith("build_")


def test_what_the_build_answers():
    from rag_amd import _build
    ask = lambda *a: subprocess.run([sys.executable, "-m", "rag_amd._build", *a], cwd=ROOT, capture_output=True, text=True, check=True).stdout.split()   # noqa: E731
    for src in _build.SOURCES:
        flags = ask("--flags", src)
        assert flags == _build.FLAGS + _build.FILE_FLAGS.get(src, [])
        i = flags.index("-packed-fp32-ops")
        assert flags[i - 3:i] == ["-Xclang", "-target-feature", "-Xclang"]
    assert ask("--objects") == [f"build/obj/{s[:-4]}.o" for s in _build.SOURCES]
    assert ask("--objects", "encoder.hip") == [o for o in ask("--objects") if o != "build/obj/encoder.o"]
