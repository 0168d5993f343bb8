"""Where built kernels read a matrix product's result before the matrix unit has to have written it.

A vector or memory instruction that reads the result of a v_mfma must stand a number of wait states behind it; the hardware does
not hold it back. The compiler keeps the distance for every instruction that it knows, but it does not look into inline assembly. So the
built code objects are looked through: from each product along every path (branches taken and not), an instruction counts one state and
s_nop n counts n + 1. Nor does it look into reads of a register that an index chooses at run time (s_set_gpr_idx_on): those may be of any.
"""
from __future__ import annotations

import glob
import os
import re
import subprocess

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
# wait states between a product and the first read of its result (what the compiler itself leaves in front of a v_max3_f32)
STATES = {"32x32x16_bf16": 12, "32x32x16_f16": 12, "16x16x32_bf16": 8, "16x16x32_f16": 8, "16x16x4_f32": 10, "32x32x2_f32": 18}
REGISTER = re.compile(r"\b([va])(?:(\d+)|\[(\d+):(\d+)\])")
READS = re.compile(r"(v_|global_store|buffer_store|flat_store|scratch_store|ds_)")


def registers(text):
    out = set()
    for kind, one, first, last in REGISTER.findall(text):
        out.update((kind, i) for i in (range(int(one), int(one) + 1) if one else range(int(first), int(last) + 1)))
    return out


def functions(library, folder):
    """(name, [(address, instruction, branch target or None)]) of every function with a matrix product."""
    link = os.path.join(folder, "lib.so")  # the code objects are written beside the file that they come from
    os.symlink(os.path.abspath(library), link)
    subprocess.run([OBJDUMP, "--offloading", link], check=True, stdout=subprocess.DEVNULL)
    for path in sorted(glob.glob(link + ".*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], check=True, stdout=subprocess.PIPE, text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
            head = re.match(r"[0-9a-f]{16} <(\S+)>:\n", part)
            if head is None or "v_mfma" not in part:
                continue
            code, begin = [], None
            for line in part[head.end():].splitlines():
                op, _, tail = line.partition("//")
                at = re.match(r"\s*([0-9A-F]+):", tail)
                if at is None:
                    continue
                at = int(at.group(1), 16)
                begin = at if begin is None else begin
                to = re.search(r"<" + re.escape(head.group(1)) + r"(?:\+0x([0-9a-f]+))?>", tail)
                code.append((at, op.strip(), begin + int(to.group(1) or "0", 16) if to else None))
            yield head.group(1), code


def early_reads(code, by_index_only=False):
    """(product, reading instruction, states between them, states needed) of a function's code."""
    place = {at: i for i, (at, _, _) in enumerate(code)}
    found = set()
    for i, (_, product, _) in enumerate(code):
        if not product.startswith("v_mfma"):
            continue
        name, args = product.split(None, 1)
        need = STATES[name[len("v_mfma_f32_"):]]
        paths, seen = [(i + 1, 0, frozenset(registers(args.split(",")[0])), False)], {}
        while paths:
            j, states, live, indexed = paths.pop()
            if j >= len(code) or states >= need or not live or seen.get((j, live, indexed), need) <= states:
                continue
            seen[j, live, indexed] = states
            _, op, to = code[j]
            name, _, args = op.partition(" ")
            if name.startswith("s_set_gpr_idx"):
                indexed = name == "s_set_gpr_idx_on"
            if READS.match(name) and not name.startswith("v_mfma"):
                written, _, read = args.partition(",") if name.startswith("v_") else ("", "", args)
                if indexed or not by_index_only and registers(read) & live:
                    found.add((product, op, states, need))
            if name.startswith("v_"):
                live = live - registers(args.partition(",")[0])
            if name == "s_endpgm":
                continue
            if to is not None:
                paths.append((place[to], states + 1, live, indexed))
                if name == "s_branch":
                    continue
            paths.append((j + 1, states + (int(args, 0) + 1 if name == "s_nop" else 1), live, indexed))
    return sorted(found)
