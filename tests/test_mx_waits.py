"""The waits of the MXFP8 kernel for few rows, checked in the built device code:
it counts the loads and copies that may still be in flight when it reads the X
rows of a step, which holds as long as the compiler keeps every one of them, on
its side of the wait."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
SKINNY = re.compile(r"mx_skinny_kernelILb([01])ELi(\d+)ELi(\d+)ELi(\d+)E")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{(X tiles, W tiles): instructions} of the kernel's instances in libpa.so."""
    lib = os.path.join(ROOT, "vllm-lite_amd", "libpa.so")
    if not os.path.exists(lib) or not os.path.exists(OBJDUMP):
        pytest.skip("no built library or no disassembler")
    d = tmp_path_factory.mktemp("mx_waits")
    shutil.copy(lib, d / "libpa.so")
    subprocess.run([OBJDUMP, "--offloading", "libpa.so"], cwd=d, check=True, capture_output=True)
    out = []
    for name in sorted(os.listdir(d)):
        if "gfx950" not in name:
            continue
        r = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", name], cwd=d, check=True,
                           capture_output=True, text=True)
        insns = None
        for line in r.stdout.splitlines():
            if line.endswith(">:"):
                m = SKINNY.search(line)
                insns = [] if m else None
                if m:
                    out.append((int(m[2]), int(m[3]), insns))
            elif insns is not None and line.startswith("\t"):
                insns.append(line.split("//")[0].strip())
    assert out, "no such kernel in libpa.so"
    return out


def test_every_counted_load_is_issued(kernels):
    """In front of each wait for all but one step's loads and copies, the last
    of them are one step's: its copies of X and then its loads."""
    for mt, nt, insns in kernels:
        copies, loads = 2 * mt, 3 * nt + mt
        issued, waits = [], 0
        for i in insns:
            if i.startswith(("global_load", "buffer_load", "flat_load")):
                issued.append("_lds_" in i)
            elif i.startswith(("global_store", "scratch_", "buffer_store")):
                issued.append(None)
            elif re.search(rf"vmcnt\({copies + loads}\)", i):
                waits += 1
                assert issued[-copies - loads:] == [True] * copies + [False] * loads, (mt, nt)
        assert waits >= 3, (mt, nt)  # two steps a turn of the loop, and the last but one
