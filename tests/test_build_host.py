"""The build's flags (no GPU, nothing is compiled)."""
import glob
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "grove_amd", "csrc")
NO_PACKED = "-Xclang -target-feature -Xclang -packed-fp32-ops"

needs_make = pytest.mark.skipif(not shutil.which("make"), reason="make not installed")


@needs_make
def test_a_changed_makefile_rebuilds_every_object():
    """Otherwise a tree that was built before a change of flags keeps objects of the old ones."""
    out = subprocess.run(["make", "-C", CSRC, "-n", "-W", "Makefile"], check=True, capture_output=True, text=True).stdout
    built = set(re.findall(r"-c (\w+)\.hip", out))
    assert built == {os.path.basename(f)[:-4] for f in glob.glob(os.path.join(CSRC, "*.hip"))}


@needs_make
def test_flags_leave_packed_arithmetic_off():
    out = subprocess.run(["make", "-s", "-C", CSRC, "flags"], check=True, capture_output=True, text=True).stdout
    assert NO_PACKED in out and "--offload-arch=gfx950" in out


def test_scripts_compile_with_the_same_flags():
    """Every command that makes device code takes the Makefile's flags or leaves packed arithmetic off itself."""
    bad = []
    for path in glob.glob(os.path.join(ROOT, "tools", "**", "*.*"), recursive=True):
        if not path.endswith((".sh", ".py", ".hip")):
            continue
        for n, line in enumerate(open(path), 1):
            if re.search(r"hipcc\b.* -(c|S|O3)\b", line) and NO_PACKED not in line and not re.search(r"\$FLAGS|make -s -C grove_amd/csrc flags", line):
                bad.append(f"{os.path.relpath(path, ROOT)}:{n}: {line.strip()}")
    assert not bad, "\n".join(bad)
