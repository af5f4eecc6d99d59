"""The built kernels wait for their matrix products: on every path, the wait states that gfx950 asks for
lie between a matrix instruction and the first other use of its result.  The hardware does not
hold such a use back (it reads what was there before), and the compiler (ROCm 7.2) has left waits
out where a branch follows on the products and paths of different length meet."""
import os
import re
import struct
import subprocess
from pathlib import Path

import pytest

LIB = Path(__file__).resolve().parent.parent / "onnx_runtime_dart_amd" / "lib" / "libmigemm.so"
OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")


def wait_states(op, rest):
    """Wait states from a matrix instruction to another's use of its result: what the compiler
    puts between the two in straight code."""
    if "f8f6f4" in op:
        # Formats 0 and 1 are of 8 bits, 2 to 4 of 6 and 4.
        small = all(int(m[1]) >= 2 if (m := re.search(name + r":(\d)", rest)) else False
                    for name in ("cbsz", "blgp"))
        return {"32x32x64": 16, "16x16x128": 12}[op.split("_")[-2]] - (4 if small else 0)
    return {"v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_32x32x16_f16": 12,
            "v_mfma_i32_32x32x32_i8": 12, "v_mfma_f32_32x32x2_f32": 16}[op]


def code_objects(lib):
    """The gfx950 code objects inside a library."""
    data, at = lib.read_bytes(), 0
    while (at := data.find(b"__CLANG_OFFLOAD_BUNDLE__", at)) >= 0:
        p = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            offset, size, n = struct.unpack_from("<QQQ", data, p)
            if data[p + 24:p + 24 + n].endswith(b"gfx950") and size:
                yield data[at + offset:at + offset + size]
            p += 24 + n
        at += 24


LINE = re.compile(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]{12}):")
TARGET = re.compile(r"<.*\+0x([0-9a-f]+)>|<([^+>]*)>")
RANGE = re.compile(r"^([va])\[(\d+):(\d+)\]|^([va])(\d+)$")


def registers(text):
    """Vector registers of an operand."""
    m = RANGE.match(text.lstrip("-|").rstrip("|"))
    if not m:
        return frozenset()
    if m[1]:
        return frozenset((m[1], i) for i in range(int(m[2]), int(m[3]) + 1))
    return frozenset([(m[4], int(m[5]))])


def kernels(text):
    """(name, first address, instructions (op, operands, address, the rest of the line)) of a disassembly."""
    name, start, out = None, 0, []
    for line in text.splitlines():
        if m := re.match(r"^([0-9a-f]{16}) <(.*)>:$", line):
            if name:
                yield name, start, out
            name, start, out = m[2], int(m[1], 16), []
        elif name and (m := LINE.match(line)):
            out.append((m[1], m[2], int(m[3], 16), line[m.end():]))
    if name:
        yield name, start, out


def early_uses(start, code):
    """Instructions that use a product's result before it is there, over all paths."""
    at = {a: i for i, (_, _, a, _) in enumerate(code)}
    ends, first = {}, {0}
    for i, (op, _, a, rest) in enumerate(code):
        if op.startswith(("s_cbranch", "s_branch")):
            to = at[start + int(TARGET.search(rest)[1] or "0", 16)]
            ends[i] = [to] if op == "s_branch" else [to, i + 1]
            first |= {to, i + 1}
        elif op == "s_endpgm":
            ends[i] = []
            first.add(i + 1)
    first = sorted(i for i in first if i < len(code))
    last = {b: (first[n + 1] if n + 1 < len(first) else len(code)) - 1 for n, b in enumerate(first)}
    parts = [[registers(x.split(" ")[0]) for x in re.split(r",\s*", text)]
             if op.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")) else []
             for op, text, _, _ in code]
    into = {b: {} for b in first}  # pending registers and their wait states
    seen, work, bad = set(), [0], set()
    while work:
        b = work.pop()
        seen.add(b)
        wait = dict(into[b])
        for i in range(b, last[b] + 1):
            op, text, _, _ = code[i]
            regs = parts[i]
            if regs and wait:
                # (A product may go on to the next as its sum at once.)
                used = regs[1:3] if op.startswith("v_mfma") else regs
                if any(r in wait for part in used for r in part):
                    bad.add(i)
            n = int(text, 0) + 1 if op == "s_nop" else 1
            wait = {r: w - n for r, w in wait.items() if w > n}
            if op.startswith("v_mfma"):
                wait.update((r, wait_states(op, text)) for r in regs[0])
        for to in ends.get(last[b], [last[b] + 1]):
            if to >= len(code):
                continue
            more = {r: w for r, w in wait.items() if into[to].get(r, 0) < w}
            if more or to not in seen:
                into[to].update(more)
                if to not in work:
                    work.append(to)
    return [f"{code[i][0]} {code[i][1]}" for i in sorted(bad)]


def disassembled(objects, folder):
    for n, obj in enumerate(objects):
        path = folder / f"{n}.co"
        path.write_bytes(obj)
        yield subprocess.run([str(OBJDUMP), "-d", str(path)], capture_output=True, text=True,
                             check=True).stdout


@pytest.mark.skipif(not OBJDUMP.exists(), reason="no llvm-objdump")
def test_products_are_waited_for(tmp_path):
    lib = Path(os.environ.get("MIGEMM_LIBRARY", LIB))
    bad, count = {}, 0
    for text in disassembled(code_objects(lib), tmp_path):
        for name, start, code in kernels(text):
            if any(op.startswith("v_mfma") for op, _, _, _ in code):
                count += 1
                if early := early_uses(start, code):
                    bad[name] = early[:4]
    assert count > 50  # kernels with matrix products
    assert not bad, bad


def listing(*lines):
    code = [(x.split(" ", 1) + [""])[:2] for x in lines]
    return [(op, text, 4 * i, f" <k+0x{4 * int(text):x}>" if "branch" in op else "")
            for i, (op, text) in enumerate(code)]


def test_paths_that_meet():
    # The wait is there on the long way round (3, 4) and missing on the short one.
    mfma, use = "v_mfma_f32_16x16x32_f16 v[0:3], v[4:7], v[8:11], 0", "v_add_f32_e32 v20, v3, v21"
    assert early_uses(0, listing(mfma, "s_nop 7", use, "s_endpgm")) == []
    assert early_uses(0, listing(mfma, "s_nop 6", use, "s_endpgm")) == [use]
    code = [mfma, "s_cbranch_vccz 4", "s_nop 1", "s_branch 5", "s_nop 7", use, "s_endpgm"]
    assert early_uses(0, listing(*code)) == [use]
    code[2] = "s_nop 5"
    assert early_uses(0, listing(*code)) == []
    loop = ["s_nop 0", use, mfma, "s_cbranch_scc1 0", "s_endpgm"]
    assert early_uses(0, listing(*loop)) == [use]
