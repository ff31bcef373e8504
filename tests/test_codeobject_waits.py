"""CPU test of the built gfx950 code objects: the wait states in front of every
vector-memory instruction.  The kernels copy to LDS in inline asm
(``lds_dma_b128``), and hipcc's hazard recognizer does not look into inline asm: a
buffer descriptor whose registers were written by a vector instruction
(``v_readfirstlane``, ``v_readlane``) needs five wait states before the copy that
reads it, or the copy takes what the registers held before.  The libraries
built here are disassembled and every path through every kernel is followed."""

import os
import re
import subprocess
import tempfile

import pytest

from harp_amd import _lib
from test_codeobject import LLVM, MAGIC, TARGET

WAIT_STATES = 5  # a vector instruction's write of an SGPR -> a vector-memory instruction's read of it


def disassembly(lib):
    """The text of every code object in the library's .hip_fatbin section."""
    with tempfile.TemporaryDirectory() as d:
        fb = os.path.join(d, "fatbin")
        subprocess.run([f"{LLVM}/llvm-objcopy", f"--dump-section=.hip_fatbin={fb}", str(lib), os.devnull], check=True,
                       capture_output=True)
        data = open(fb, "rb").read()
        starts = [m.start() for m in re.finditer(re.escape(MAGIC), data)]
        for i, st in enumerate(starts):
            part, co = os.path.join(d, f"b{i}"), os.path.join(d, f"co{i}.o")
            with open(part, "wb") as f:
                f.write(data[st:starts[i + 1] if i + 1 < len(starts) else len(data)])
            subprocess.run([f"{LLVM}/clang-offload-bundler", "--unbundle", "--type=o", f"--input={part}",
                            f"--targets={TARGET}", f"--output={co}"], check=True, capture_output=True)
            yield subprocess.run([f"{LLVM}/llvm-objdump", "-d", "--no-show-raw-insn", co], check=True,
                                 capture_output=True, text=True).stdout


def kernels(text):
    """(name, [(address, instruction, branch target or None)]) of every function of a listing."""
    name, ins = None, []
    for line in text.splitlines():
        m = re.match(r"([0-9a-f]+) <(\S+)>:", line)
        if m:
            if ins:
                yield name, ins
            name, base, ins = m.group(2), int(m.group(1), 16), []
            continue
        m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):(.*)", line)
        if m:
            target = re.search(r"<[^+>]+(?:\+0x([0-9a-f]+))?>", m.group(3))
            ins.append((int(m.group(2), 16), m.group(1), base + int(target.group(1) or "0", 16) if target else None))
    if ins:
        yield name, ins


def scalars(operand):
    """The numbers of the SGPRs that an operand names."""
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return range(int(m.group(1)), int(m.group(2)) + 1)
    m = re.fullmatch(r"s(\d+)", operand)
    return range(int(m.group(1)), int(m.group(1)) + 1) if m else ()


def vmem(op):
    return op.startswith(("buffer_", "global_", "flat_", "scratch_"))


def short_waits(ins):
    """(address, instruction, wait states) of the vector-memory instructions that read an SGPR too early.  The
    state in front of an instruction: how many wait states ago a vector instruction wrote each SGPR, the
    shortest over all paths (those WAIT_STATES or more ago are left out)."""
    at = {a: i for i, (a, _, _) in enumerate(ins)}
    before = [None] * len(ins)
    before[0], todo, found = {}, [0], {}
    while todo:
        i = todo.pop()
        ago = before[i]
        while True:
            addr, text, target = ins[i]
            op, _, rest = text.partition(" ")
            operands = re.findall(r"s\[\d+:\d+\]|\bs\d+\b", rest)
            if vmem(op):
                for r in (r for o in operands for r in scalars(o)):
                    if r in ago:
                        found[addr] = (addr, text, min(ago[r], found.get(addr, (0, 0, WAIT_STATES))[2]))
            steps = int(rest, 0) + 1 if op == "s_nop" else 1
            after = {r: n + steps for r, n in ago.items() if n + steps < WAIT_STATES}
            if op.startswith("v_"):
                first = rest.split(",")[0].strip()
                for r in scalars(first):
                    after[r] = 0
                if "," in rest and re.match(r"v_\S+_co_", op):  # (the carry goes to the second operand)
                    for r in scalars(rest.split(",")[1].strip()):
                        after[r] = 0
            follow = []
            if op in ("s_branch",) or op.startswith("s_cbranch"):
                follow.append(at[target])
            if op not in ("s_branch", "s_endpgm", "s_setpc_b64") and i + 1 < len(ins):
                follow.append(i + 1)
            onward = []
            for j in follow:
                if before[j] is None:
                    before[j] = dict(after)
                    onward.append(j)
                else:
                    less = {r: n for r, n in after.items() if n < before[j].get(r, WAIT_STATES)}
                    if less:
                        before[j].update(less)
                        onward.append(j)
            if not onward:
                break
            todo.extend(onward[1:])
            i = onward[0]
            ago = before[i]
    return list(found.values())


def test_the_check_sees_a_short_wait():
    def listing(lines):
        return [(4 * i, t, None) for i, t in enumerate(lines)]

    copy = ["s_mov_b32 m0, s9", "s_nop 0", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds", "s_endpgm"]
    assert [f[2] for f in short_waits(listing(["v_readfirstlane_b32 s4, v0", *copy]))] == [2]
    assert [f[2] for f in short_waits(listing(["v_cmp_gt_i32_e64 s[6:7], s0, v0", "s_and_b32 s5, s5, s2", *copy]))] == [3]
    assert not short_waits(listing(["v_readfirstlane_b32 s4, v0", "s_nop 2", *copy]))
    assert not short_waits(listing(["v_readfirstlane_b32 s9, v0", *copy]))
    # around a loop: the write at its end is before the copy at its start
    loop = [(0, "s_nop 7", None), (4, copy[2], None), (8, "v_readlane_b32 s7, v9, 3", None),
            (12, "s_cbranch_scc0 65533", 4), (16, "s_endpgm", None)]
    assert [f[2] for f in short_waits(loop)] == [1]


@pytest.mark.skipif(not os.path.exists(f"{LLVM}/llvm-objdump"), reason="ROCm LLVM tools not installed")
@pytest.mark.parametrize("lib", [_lib.ABI_LIB, _lib.KERNELS / "libharp_bench_probe.so"],
                         ids=["libharp_ra", "libharp_bench_probe"])
def test_descriptors_are_settled_before_the_copies_that_read_them(lib):
    if not lib.exists():
        pytest.skip(f"{lib} not built")
    seen, copies, bad = 0, 0, []
    for text in disassembly(lib):
        for name, ins in kernels(text):
            seen += 1
            copies += sum(" lds" in t for _, t, _ in ins)
            bad += [(name, *f) for f in short_waits(ins)]
    assert seen and (copies or lib != _lib.ABI_LIB)
    assert not bad, f"{len(bad)} short waits in {sorted({b[0] for b in bad})}: {bad[:5]}"
