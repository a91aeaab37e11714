"""The matrix instructions' results that hand-written instructions read, in the built
device code: a vector instruction may read a result of v_mfma no sooner than 19 wait
states after it (16 passes; fewer need less), and the compiler, which adds them before its
own instructions, sees into no inline assembly (v_max3_f32 of the tiled attention)."""
import heapq
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
STATES = 19


def registers(operand):
    m = re.match(r"-?\|?v(?:\[(\d+):(\d+)\]|(\d+))\|?$", operand)
    if not m:
        return frozenset()
    first = int(m[1] or m[3])
    return frozenset(range(first, int(m[2] or first) + 1))


def functions(text):
    """[(name, [(address, mnemonic, operands, branch target)])]"""
    out = []
    for line in text.splitlines():
        m = re.match(r"([0-9a-f]+) <(.*)>:", line)
        if m:
            out.append((m[2], int(m[1], 16), []))
            continue
        insn, _, note = line.partition("//")
        m = re.match(r"\s*([0-9A-F]+):", note)
        if not line.startswith("\t") or not m:
            continue
        name, _, rest = insn.strip().partition(" ")
        t = re.search(r"<[^>]*?(?:\+0x([0-9a-f]+))?>\s*$", note)
        target = out[-1][1] + int(t[1] or "0", 16) if t else None
        out[-1][2].append((int(m[1], 16), name, [x.strip() for x in rest.split(",")], target))
    return [(name, code) for name, _, code in out]


def nearest(code):
    """The fewest wait states, below STATES, between a v_mfma and a v_max3_f32 that reads
    its result, over all paths; None if there are none."""
    index = {x[0]: i for i, x in enumerate(code)}
    best = None
    for i, (_, name, ops, _) in enumerate(code):
        if not name.startswith("v_mfma") or not registers(ops[0]):
            continue
        queue, seen = [(0, i + 1, registers(ops[0]))], set()
        while queue:
            states, at, live = heapq.heappop(queue)
            if states >= STATES or at >= len(code) or (at, live) in seen:
                continue
            seen.add((at, live))
            _, name, ops, target = code[at]
            if name == "v_max3_f32" and live & frozenset().union(*map(registers, ops[1:])):
                best = states if best is None else min(best, states)
                continue
            if name.startswith("v_"):
                live = live - registers(ops[0])  # overwritten
            if not live or name == "s_endpgm":
                continue
            states += int(ops[0], 0) + 1 if name == "s_nop" else 1
            if name.startswith("s_cbranch") or name == "s_branch":
                if target in index:
                    heapq.heappush(queue, (states, index[target], live))
            if name != "s_branch":
                heapq.heappush(queue, (states, at + 1, live))
    return best


def test_results_are_read_late_enough(tmp_path):
    lib = os.path.join(ROOT, "vllm-lite_amd", "libpa.so")
    if not os.path.exists(lib) or not os.path.exists(OBJDUMP):
        pytest.skip("no built library or no disassembler")
    shutil.copy(lib, tmp_path / "libpa.so")
    subprocess.run([OBJDUMP, "--offloading", "libpa.so"], cwd=tmp_path, check=True,
                   capture_output=True)
    found = 0
    for name in sorted(os.listdir(tmp_path)):
        if "gfx950" not in name:
            continue
        r = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", name], cwd=tmp_path, check=True,
                           capture_output=True, text=True)
        for function, code in functions(r.stdout):
            if "prefill" in function and any(x[1] == "v_max3_f32" for x in code):
                found += 1
                assert nearest(code) is None, (function, nearest(code))
    assert found > 0


def test_the_search_itself():
    """Straight, around a loop, behind waits and behind an overwriting instruction."""
    def code(*insns):
        return [(4 * i, n, o.split(), t) for i, (n, o, t) in enumerate(insns)]

    mfma, read = ("v_mfma_f32_16x16x32_bf16", "v[4:7] v[0:3] v[8:11] 0", None), \
        ("v_max3_f32", "v1 v2 v6 v3", None)
    other = ("v_add_f32_e32", "v20 v21 v22", None)
    assert nearest(code(mfma, read)) == 0
    assert nearest(code(mfma, other, other, read)) == 2
    assert nearest(code(read, other, mfma, other, ("s_cbranch_scc1", "0", 0))) == 2
    assert nearest(code(mfma, ("s_nop", "10", None), read)) == 11
    assert nearest(code(mfma, ("s_nop", "15", None), ("s_nop", "3", None), read)) is None
    assert nearest(code(mfma, ("v_mov_b32_e32", "v6 v0", None), read)) is None
