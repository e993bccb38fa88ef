"""The waits between matrix instructions and what uses their results, in the kernels as built (no GPU needed).

The hardware does not hold back an instruction that uses a result too early; the compiler counts the instructions between
and fills up with s_nop.  Where two ways join it has been seen to count the longer one only, after a matrix
instruction whose result is first used behind a short condition: that use reads what the registers held before."""
import os
import re
import subprocess

import pytest

from vnpu_mi355x import load_backend
from vnpu_mi355x.runtime import BACKEND_LIB

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"

# Instructions between (an s_nop n counts n + 1): passes of 4 cycles and 4 more, for f32 operands 2 more.
WAITS = {
    "v_mfma_f32_16x16x32_f16": 8, "v_mfma_i32_16x16x64_i8": 8, "v_mfma_i32_16x16x32_i8": 8,
    "v_mfma_f32_32x32x16_bf16": 12, "v_mfma_i32_32x32x32_i8": 12,
    "v_mfma_f32_16x16x4_f32": 10, "v_mfma_f32_16x16x1_4b_f32": 10, "v_mfma_f32_32x32x1_2b_f32": 18,
}
REGISTERS = re.compile(r"\b([va])(?:(\d+)|\[(\d+):(\d+)\])")


def registers(text):
    return {(m[1], n) for m in REGISTERS.finditer(text) for n in range(int(m[2] or m[3]), int(m[2] or m[4]) + 1)}


def kernels(listing):
    """(name, blocks) of each function; a block is (instructions, blocks that may follow)."""
    for part in re.split(r"^<(?=[^L]|L\D)", listing, flags=re.M)[1:]:
        name, _, body = part.partition(">:")
        if "v_mfma" not in body:
            continue
        blocks, labels = [[]], {}
        for line in body.split("\n"):
            line = line.split("//")[0].strip()
            if m := re.match(r"<(L\d+)>:", line):
                blocks.append([])
                labels[m[1]] = len(blocks) - 1
            elif line and re.match(r"[a-z]\w+", line):
                blocks[-1].append(line)
                if line.startswith(("s_branch", "s_cbranch", "s_endpgm", "s_setpc")):
                    blocks.append([])
        follow = []
        for i, block in enumerate(blocks):
            last = block[-1].split() if block else [""]
            follow.append([labels[last[1]]] if last[0].startswith(("s_branch", "s_cbranch")) else [])
            if not last[0].startswith(("s_branch", "s_endpgm", "s_setpc")) and i + 1 < len(blocks):
                follow[-1].append(i + 1)
        yield name, list(zip(blocks, follow))


def early(blocks):
    """(matrix instruction, first use, instructions between) where a way between them is too short."""
    for start, (block, _) in enumerate(blocks):
        for at, line in enumerate(block):
            if not line.startswith("v_mfma"):
                continue
            op, _, operands = line.partition(" ")
            need, result = WAITS[op], registers(operands.split(",")[0])
            ways, seen = [(start, at + 1, 0)], {}
            while ways:
                b, i, count = ways.pop()
                if seen.get((b, i), need) <= count:
                    continue
                seen[b, i] = count
                lines, follow = blocks[b]
                while i < len(lines) and count < need:
                    name, _, rest = lines[i].partition(" ")
                    if name.startswith("v_mfma"):   # as the summand it may follow at once; the same result again is a new one
                        to, *factors = rest.split(",")[:3]
                        if registers(" ".join(factors)) & result:
                            yield line, lines[i], count
                        if registers(to) & result:
                            break
                    elif name.startswith(("v_", "ds_", "buffer_", "global_", "flat_", "scratch_")) and registers(rest) & result:
                        yield line, lines[i], count
                        break
                    count += int(rest, 0) + 1 if name == "s_nop" else 1
                    i += 1
                else:
                    if count < need:
                        ways += [(f, 0, count) for f in follow]


LISTING = """
<short_way>:
	v_mfma_i32_16x16x64_i8 v[0:3], v[8:11], v[12:15], 0
	s_cbranch_vccnz L1
	s_nop 15
<L1>:
	v_add_u32_e32 v4, v3, v4
	s_endpgm
<long_way>:
	v_mfma_i32_16x16x64_i8 v[0:3], v[8:11], v[12:15], 0
	v_mfma_i32_16x16x64_i8 v[0:3], v[8:11], v[12:15], v[0:3]
	s_nop 6
	s_cbranch_vccnz L3
<L2>:
	s_nop 0
<L3>:
	v_add_u32_e32 v4, v3, v4
	s_endpgm
<as_a_factor>:
	v_mfma_i32_16x16x64_i8 v[0:3], v[8:11], v[12:15], 0
	v_mfma_i32_16x16x64_i8 v[4:7], v[0:3], v[12:15], 0
	s_endpgm
"""


def test_the_count_itself():
    found = {name: [between for _, _, between in early(blocks)] for name, blocks in kernels(LISTING)}
    assert found == {"short_way": [1], "long_way": [], "as_a_factor": [0]}


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler here")
def test_results_are_waited_for_on_every_way(tmp_path):
    load_backend()
    library = tmp_path / "libvnpu.so"
    library.symlink_to(os.path.realpath(BACKEND_LIB))
    subprocess.run([OBJDUMP, "--offloading", str(library)], cwd=tmp_path, check=True, capture_output=True)
    count, bad = 0, []
    for code in sorted(tmp_path.glob("*gfx950*")):
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--symbolize-operands", "--mcpu=gfx950", str(code)],
                                 check=True, capture_output=True, text=True).stdout
        for name, blocks in kernels(re.sub(r"^\s*[0-9a-f]+ (?=<)", "", listing, flags=re.M)):
            count += 1
            bad += [(name, *x) for x in early(blocks)]
    assert count > 100
    assert not bad, (len({b[0] for b in bad}), bad[:3])
