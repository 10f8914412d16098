"""Wait states of the hand-issued DMA, in the disassembly of the built library: a
vector-memory instruction may not read a scalar register within five wait states of
the vector instruction that wrote it.  The compiler keeps to that for the
instructions it emits, not for what stands inside inline assembly."""
import os
import re
import shutil
import subprocess

import pytest
from test_split_resources import _code_objects

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
WAIT = 5


def _scalars(operand):
    """Numbers of the scalar registers that an operand names."""
    one = re.fullmatch(r"s(\d+)|s\[(\d+):(\d+)\]", operand)
    if not one:
        return range(106, 108) if operand == "vcc" else ()
    if one[1]:
        return (int(one[1]),)
    return range(int(one[2]), int(one[3]) + 1)


def _violations(lines):
    """(kernel, instruction, wait states) of each read that comes too early, and how
    many vector-memory instructions read scalar registers at all."""
    bad, seen, name, at, written = [], 0, "", 0, {}
    for line in lines:
        label = re.match(r"[0-9a-f]+ <(.+)>:", line)
        if label:
            name, written = label[1], {}
            continue
        text = line.split("//")[0].strip()
        if not text or not line[0].isspace():
            continue
        op, _, rest = text.partition(" ")
        operands = [o.strip().split(" ")[0] for o in rest.split(",")]
        if op.startswith(("buffer_", "global_", "flat_", "scratch_")):
            read = [s for o in operands for s in _scalars(o)]
            seen += bool(read)
            waits = min((at - written[s] for s in read if s in written), default=WAIT)
            if waits < WAIT:
                bad.append((name, text, waits))
        at += int(operands[0], 0) + 1 if op == "s_nop" else 1
        # the first operand is the destination, and a carry the second
        carry = "_co_" in op or op.startswith(("v_div_scale", "v_mad_u64", "v_mad_i64"))
        for o in operands[:1 + carry]:
            for s in _scalars(o):
                if op.startswith("v_"):
                    written[s] = at
                else:
                    written.pop(s, None)
    return bad, seen


def test_scan_finds_what_it_looks_for():
    text = """0000 <kernel>:
\tv_readfirstlane_b32 s5, v1                                 // 0
\ts_add_u32 m0, s9, 0x400                                    // 8
\ts_nop 0                                                    // 10
\tbuffer_load_dwordx4 v2, s[4:7], 0 offen lds                // 18
\tv_readfirstlane_b32 s5, v1                                 // 20
\ts_add_u32 m0, s9, 0x400                                    // 28
\ts_nop 3                                                    // 30
\tbuffer_load_dwordx4 v2, s[4:7], 0 offen lds                // 38
\tv_readfirstlane_b32 s5, v1                                 // 40
\ts_mov_b32 s5, s8                                           // 48
\tglobal_load_dword v1, v2, s[4:5]                           // 50
""".splitlines()
    assert _violations(text) == ([("kernel", "buffer_load_dwordx4 v2, s[4:7], 0 offen lds", 2)], 3)


def test_dma_waits_for_its_scalar_operands(tmp_path):
    from ozaki_triton_amd import build
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    kernels = 0
    for n, obj in enumerate(_code_objects(build.LIB_PATH)):
        if b"TileShape" not in obj:
            continue
        path = tmp_path / str(n)
        path.write_bytes(obj)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], capture_output=True,
                              text=True, check=True).stdout
        bad, seen = _violations(text.splitlines())
        assert seen > 100
        kernels += 1
        assert not bad, (len(bad), bad[:4])
    assert kernels == 2      # grouped products, orthogonalisation
