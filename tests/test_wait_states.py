"""No-GPU check of the built kernels of the delta rule: on every path from a matrix instruction to the first use of its result there are the wait states that the hardware needs.  The compiler
keeps them by itself, except round a short conditional block between the two (see delta_chunk.hip), where a use would read the registers as they were before."""
import os
import re
import shutil
import struct
import subprocess

import pytest
from pooled_amd import build

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
# wait states from a matrix instruction of gfx950 to a vector or memory instruction, or to another one's factors, that reads its result; as the compiler itself counts them: passes + 4, f32 passes + 2
NEEDED = {"v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x4_f32": 10}


def code_object(path):
    """The gfx950 part of a host object's offload bundle."""
    data = open(path, "rb").read()
    at = data.index(b"__CLANG_OFFLOAD_BUNDLE__")
    count, pos = struct.unpack_from("<Q", data, at + 24)[0], at + 32
    for _ in range(count):
        offset, size, n = struct.unpack_from("<3Q", data, pos)
        name = data[pos + 24:pos + 24 + n]
        pos += 24 + n
        if b"gfx950" in name:
            return data[at + offset:at + offset + size]
    raise AssertionError("no gfx950 code in " + path)


def functions(text):
    """name -> [(address, instruction, [operands], branch target)]"""
    out = {}
    for line in text.splitlines():
        m = re.match(r"^([0-9a-f]+) <(\w+)>:", line)
        if m:
            out[m[2]] = code = []
            base = int(m[1], 16)
            continue
        m = re.match(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):", line)
        if not m:
            continue
        t = re.search(r"<\w+\+0x([0-9a-f]+)>\s*$", line)
        code.append((int(m[3], 16), m[1], [o.strip() for o in m[2].split(",")], base + int(t[1], 16) if t else None))
    return out


def registers(operand):
    m = re.match(r"^-?\|?([av])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.match(r"^-?\|?([av])(\d+)\b", operand)
    return {(m[1], int(m[2]))} if m else set()


def shortest(code):
    """[(matrix instruction, wait states, its use)]: the fewest on any path, for every use"""
    place = {c[0]: i for i, c in enumerate(code)}
    before = [[] for _ in code]
    for i, (_, op, _, target) in enumerate(code):
        if op.startswith("s_cbranch") or op == "s_branch":
            before[place[target]].append(i)
        if op not in ("s_branch", "s_endpgm", "s_setpc_b64") and i + 1 < len(code):
            before[i + 1].append(i)
    store = ("global_store", "ds_write", "buffer_store", "flat_store", "s_")
    found = []
    for i, (_, op, args, _) in enumerate(code):
        if op.startswith("s_"):
            continue
        read = args if op.startswith(store) or op.startswith(("v_fmac", "v_dot", "v_permlane")) else args[1:3] if op.startswith("v_mfma") else args[1:]
        for reg in set().union(*map(registers, read)) if read else ():
            seen, todo = {}, [(p, 0) for p in before[i]]
            while todo:
                j, d = todo.pop()
                if d > 24 or seen.get(j, 99) <= d:
                    continue
                seen[j] = d
                _, o, b, _ = code[j]
                if not o.startswith(store) and b and reg in registers(b[0]):
                    if o.startswith("v_mfma"):
                        found.append((o, d, "%s %s" % (op, ", ".join(args))))
                    continue
                step = int(b[0], 0) + 1 if o == "s_nop" else 1
                todo += [(p, d + step) for p in before[j]]
    return found


def disassembled(stem, tmp_path):
    obj = os.path.join(build.LIBDIR, stem + ".o")
    if not (os.path.exists(OBJDUMP) and os.path.exists(obj)):
        pytest.skip("llvm-objdump or the built object is missing")
    elf = tmp_path / (stem + ".co")
    elf.write_bytes(code_object(obj))
    return functions(subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", str(elf)], capture_output=True, text=True, check=True).stdout)


def test_chunked_delta_rule(tmp_path):
    kernels = {n: c for n, c in disassembled("delta_chunk", tmp_path).items() if "kernel" in n}
    assert len(kernels) == 6
    for name, code in kernels.items():
        uses = shortest(code)
        assert len(uses) > 50 and all(op in NEEDED for op, _, _ in uses), name
        low = min(uses, key=lambda u: u[1] - NEEDED[u[0]])
        print(name, len(uses), low)
        assert low[1] >= NEEDED[low[0]], "%s: %d wait states behind %s in front of %s" % (name, low[1], low[0], low[2])


def test_the_check_sees_a_path_round_a_block():
    text = """0000000000001000 <k>:
	v_mfma_f32_16x16x32_f16 v[0:3], v[8:11], v[12:15], 0       // 000000001000: 00
	s_cbranch_scc0 3                                           // 000000001008: 00 <k+0x14>
	s_nop 6                                                    // 00000000100C: 00
	v_add_f32_e32 v4, v0, v0                                   // 000000001010: 00
	v_mul_f32_e32 v5, s0, v3                                   // 000000001014: 00
	s_endpgm                                                   // 000000001018: 00
"""
    uses = dict((u, d) for _, d, u in sorted(shortest(functions(text)["k"]), key=lambda f: -f[1]))
    assert uses == {"v_add_f32_e32 v4, v0, v0": 8, "v_mul_f32_e32 v5, s0, v3": 1}
