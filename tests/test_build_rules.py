"""The build's rules name every header that an object's source includes, so that an edit to one rebuilds
all objects that were made with it (CPU)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "needle_amd", "csrc")


def headers_of(path, seen):
    """The repository's own headers that a source includes, and those that they include."""
    with open(path) as f:
        names = re.findall(r'^\s*#\s*include\s+"([^"]+)"', f.read(), re.M)
    for name in names:
        for d in (os.path.dirname(path), os.path.join(ROOT, "include")):
            at = os.path.realpath(os.path.join(d, name))
            if os.path.exists(at) and at not in seen:
                seen.add(at)
                headers_of(at, seen)
    return seen


@pytest.mark.skipif(not shutil.which("make"), reason="make not installed")
def test_objects_depend_on_what_their_sources_include():
    # (-r, -R: no rules and variables of make's own)
    rules = subprocess.run(["make", "-C", CSRC, "-pnqrR", "--no-print-directory"],
                           capture_output=True, text=True).stdout
    needs = {}
    for target, rest in re.findall(r"^([^\s#:=]+):(?!=)([^=\n]*)$", rules, re.M):
        needs.setdefault(target, set()).update(
            os.path.realpath(os.path.join(CSRC, x)) for x in rest.split())
    sources = sorted(x for x in os.listdir(CSRC) if x.endswith(".hip"))
    assert sources
    for x in sources:
        missing = headers_of(os.path.join(CSRC, x), set()) - needs[f"_build/{x[:-4]}.o"]
        assert not missing, (x, missing)
    assert headers_of(os.path.join(CSRC, "bind.cpp"), set()) <= needs["../_native.so"]
