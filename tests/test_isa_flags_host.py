"""ISA checks of what is built (no GPU): the flags are those of the Makefile, so the code that is looked at is the code that ships. Every file
whose kernels count their own vector memory waits: a wait that hipcc adds inside such a loop drains the loads that the loop keeps in
flight (the scan of tools/isa_loop_waits.py; the unpacked epilogues of the 256-row ReLU and scaled GEMMs got such waits, 5 to 10 % of their time)."""
import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "grove_amd", "csrc")
sys.path.insert(0, os.path.join(ROOT, "tools"))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
FILES = ["gemm", "gemm_tn", "flash_attn2", "kv4"]

# instances that keep such a wait: QuickGELU at K = 1024, where the cure measured slower (tools/dev/pp_drain_ab.py), and the FP8 ones
ACCEPTED = ("gemm_nt_pp_kernelILi256ELb0ELi3E", "ELb1ELb0EEEv17grove_gemm_params")
# registers that an instance of kv4_attn_kernel spills outside its loop, by its template arguments (<128, 4>: 64 columns, two waves a SIMD)
SPILLS = {(128, 4): 7}


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    if not os.path.exists(HIPCC) or not shutil.which("make"):
        pytest.skip("hipcc or make not installed")
    flags = subprocess.run(["make", "-s", "-C", CSRC, "flags"], check=True, capture_output=True, text=True).stdout.split()
    out = tmp_path_factory.mktemp("asm")

    def one(name):
        path = str(out / (name + ".s"))
        subprocess.run([HIPCC, *flags, "-Wno-unused-command-line-argument", "-S", "--cuda-device-only", os.path.join(CSRC, name + ".hip"), "-o", path],
                       check=True, capture_output=True)
        return path
    with ThreadPoolExecutor(len(FILES)) as ex:
        return dict(zip(FILES, ex.map(one, FILES)))


def test_no_compiler_wait_in_counted_loops(asm):
    from isa_loop_waits import scan, short
    bad = []
    for name, least in zip(FILES, (30, 4, 8, 10)):
        found = scan(asm[name])
        assert len(found) >= least, f"{name}: only {len(found)} LDS-DMA loops found"
        bad += [(short(r["kernel"]), r["loop"], r["waits"][:3]) for r in found if r["waits"] and not any(a in r["kernel"] for a in ACCEPTED)]
    assert not bad, "\n".join(map(str, bad))


def test_no_packed_arithmetic(asm):
    for name, path in asm.items():
        found = re.findall(r"v_pk_(?:add|mul|fma)_f32", open(path).read())
        assert not found, (name, len(found))


def test_attention_spills(asm):
    """Spilled registers of the 4-bit attention: none, but for the instances above."""
    text = open(asm["kv4"]).read()
    seen = {}
    for name, body in re.findall(r"\.name:\s+(\S+)\n(.*?)\.wavefront_size", text, re.S):
        m = re.search(r"kv4_attn_kernelILi(\d+)ELi(\d+)E", name)
        if m:
            seen[int(m[1]), int(m[2])] = int(re.search(r"vgpr_spill_count:\s+(\d+)", body)[1])
    assert len(seen) == 11
    assert all(n <= SPILLS.get(k, 0) for k, n in seen.items()), seen
