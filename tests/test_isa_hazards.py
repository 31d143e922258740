"""Wait states in the machine code of the built library.  The compiler keeps the distances that the hardware asks for between
dependent instructions, but it does not look into inline assembly: an instruction written there, or one right behind it, can
come too early and then reads what a register held before -- now and then, as the timing of the other waves has it.  The
distances that the library's own assembly can violate are looked for in the whole code."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from ollama_amd import qmm

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(path):
    """the gfx950 code objects bundled in a shared library"""
    data = open(path, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        (count,) = struct.unpack_from("<Q", data, at + 24)
        p = at + 32
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + length]:
                yield data[at + offset:at + offset + size]
            p += 24 + length
        at = data.find(MAGIC, at + 1)


def registers(operand):
    """the vector registers that an operand names"""
    m = re.fullmatch(r"-?\|?v(\d+)\|?", operand)
    if m:
        return {int(m.group(1))}
    m = re.fullmatch(r"-?\|?v\[(\d+):(\d+)\]\|?", operand)
    return set(range(int(m.group(1)), int(m.group(2)) + 1)) if m else set()


def scalars(text):
    """the scalar registers that operands name"""
    found = {int(x) for x in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(a), int(b) + 1))
    return found


SWAP = re.compile(r"v_permlane(16|32)_swap")
DPP = re.compile(r"\b(quad_perm|row_shl|row_shr|row_ror|row_bcast|row_mirror|row_half_mirror|wave_\w+|row_newbcast)\b")


def hazards(lines):
    """(function, what is too close) for every violation; the distances of the published tables, in wait states:
    a vector register written by the vector ALU -> read by a lane swap or through a lane permutation (dpp): 2;
    a scalar register written by the vector ALU -> read by a vector memory instruction: 5;
    m0 written -> a load that goes to LDS: 1"""
    # recent: (wait states it takes, vector and scalar registers written by the vector ALU, writes m0)
    function, recent, found = None, [], []
    for line in lines:
        if line.endswith(">:"):
            function, recent = line.split("<", 1)[-1][:-2], []
            continue
        text = line.split("//")[0].strip()
        if not text or text.endswith(":"):
            continue
        op, _, rest = text.partition(" ")
        if op in ("s_branch", "s_endpgm", "s_setpc_b64"):
            recent = []
            continue
        if op == "s_nop":
            recent = (recent + [(int(rest, 0) + 1, set(), set(), False)])[-6:]
            continue
        args = [a.strip() for a in rest.split(",")]
        if args:
            args[-1] = args[-1].split(" ")[0]
        reads, need = set(), 0
        if SWAP.match(op):
            reads, need = registers(args[0]) | registers(args[1]), 2
        elif op.startswith("v_") and DPP.search(rest):
            reads, need = registers(args[1].split(" ")[0]), 2
        to_lds = "_lds_" in op or (op.startswith("buffer_load") and rest.endswith(" lds"))
        bases = scalars(rest) if op.startswith(("global_", "buffer_", "flat_", "scratch_")) else set()
        distance = 0
        for states, written, scalar, m0 in reversed(recent):
            if distance < 5 and scalar & bases:
                found.append((function, f"{text}: its base was written {distance} wait states before"))
            if distance < need and written & reads:
                found.append((function, f"{text}: its register was written {distance} wait states before"))
            if distance < 1 and m0 and to_lds:
                found.append((function, f"{text}: m0 was written right before"))
            distance += states
        written, scalar = set(), set()
        if op.startswith(("v_readlane", "v_readfirstlane", "v_cmp")):
            scalar = scalars(args[0])
        elif op.startswith("v_") and len(args) > 1:  # a carry or a scale flag
            scalar = scalars(args[1]) if re.match(r"v_(add|sub|subrev)_co|v_(addc|subb|subbrev)_co|v_div_scale|v_mad_[ui]64", op) else set()
        if op.startswith("v_") and not op.startswith(("v_cmp", "v_mfma", "v_smfma", "v_readlane", "v_readfirstlane")):
            written = registers(args[0]) | (registers(args[1]) if SWAP.match(op) else set())
        recent = (recent + [(1, written, scalar, op.startswith("s_") and args[:1] == ["m0"])])[-6:]
    return found


def test_the_check_sees_what_it_looks_for():
    code = """
0000000000001000 <f>:
\tv_mov_b32_e32 v66, v130
\tv_mov_b32_e32 v67, v132
\ts_ashr_i32 s8, s86, 31
\tv_permlane32_swap_b32_e32 v66, v67
\ts_mov_b32 m0, s4
\tglobal_load_lds_dwordx4 v1, s[0:1]
\tv_add_f32_e32 v1, v2, v3
\ts_nop 0
\tv_mov_b32_dpp v4, v1 row_shr:1 row_mask:0xf bank_mask:0xf
0000000000002000 <g>:
\tv_mov_b32_e32 v67, v132
\ts_nop 1
\tv_permlane32_swap_b32_e32 v66, v67
\ts_mov_b32 m0, s4
\ts_nop 0
\tglobal_load_lds_dwordx4 v1, s[0:1]
\tv_add_f32_e32 v1, v2, v3
\ts_nop 1
\tv_mov_b32_dpp v4, v1 row_shr:1 row_mask:0xf bank_mask:0xf
\tv_mfma_f32_16x16x32_f16 v[0:3], v[4:7], v[8:11], v[0:3]
0000000000003000 <h>:
\tv_readfirstlane_b32 s7, v109
\ts_mov_b32 m0, s4
\ts_nop 2
\tglobal_load_lds_dwordx4 v175, s[6:7]
\tv_readfirstlane_b32 s6, v109
\ts_mov_b32 m0, s4
\ts_nop 3
\tglobal_load_lds_dwordx4 v175, s[6:7]
"""
    found = hazards(code.splitlines())
    assert [f for f, _ in found] == ["f"] * 3 + ["h"]
    assert "v66, v67" in found[0][1] and "m0" in found[1][1] and "row_shr" in found[2][1] and "base was written 4" in found[3][1]


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    """(instructions of the built library, violations)"""
    if not shutil.which(OBJDUMP):
        pytest.skip("no disassembler here")
    lines, found = [], []
    for i, o in enumerate(code_objects(qmm.LIB_PATH)):
        elf = tmp_path_factory.mktemp("code") / f"{i}.elf"
        elf.write_bytes(o)
        out = subprocess.run([OBJDUMP, "-d", "--no-leading-addr", "--no-show-raw-insn", str(elf)], check=True, capture_output=True, text=True)
        lines += out.stdout.splitlines()
        found += hazards(out.stdout.splitlines())
    return lines, found


def test_registers_of_lane_swaps(built):
    lines, found = built
    assert any(SWAP.search(x) for x in lines) and any(DPP.search(x) for x in lines)  # the instructions in question are there
    found = [f for f in found if "its register" in f[1]]
    assert not found, f"{len(found)}, the first: {found[:5]}"


def test_m0_of_loads_to_lds(built):
    lines, found = built
    assert any("_load_lds_" in x for x in lines)
    found = [f for f in found if "m0" in f[1]]
    assert not found, f"{len(found)}, the first: {found[:5]}"


def test_bases_of_vector_memory(built):
    lines, found = built
    found = [f for f in found if "its base" in f[1]]
    assert not found, f"{len(found)}, the first: {found[:5]}"
