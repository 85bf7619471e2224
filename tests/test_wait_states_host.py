"""The matrix instructions written as inline assembly: the compiler does not see into them, so the wait states that it would
put between a vector instruction and an MFMA that reads its result have to be there by construction. Read off the
assembly of the kernels, over every path into each instruction."""

import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from trnblas_amd import build

WAIT_STATES = 2  # a vector ALU write of a register, then an MFMA that reads it

_REG = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")


def _registers(operand):
    """The vector and accumulation registers that an operand names."""
    return {(m[1], n) for m in _REG.finditer(operand) for n in range(int(m[2] or m[3]), int(m[2] or m[4]) + 1)}


def _parse(text):
    """{kernel: (instructions, {label: index})}: (mnemonic, operands) in order."""
    kernels, code, labels = {}, None, None
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        if not line:
            continue
        if re.match(r"^_Z\w+:$", line):
            code, labels = [], {}
            kernels[line[:-1]] = code, labels
        elif line.startswith(".Lfunc_end"):
            code = None
        elif code is not None and line.endswith(":"):
            labels[line[:-1]] = len(code)
        elif code is not None and not line.startswith("."):
            name, _, rest = line.partition(" ")
            code.append((name, [x.strip() for x in re.split(r",(?![^\[]*\])", rest)]))
    return kernels


def hazards(text, needed=WAIT_STATES):
    """(kernel, index, write, MFMA) wherever fewer than the needed wait states lie between the two on some path."""
    found = []
    for kernel, (code, labels) in _parse(text).items():
        before = [[i - 1] if i and code[i - 1][0] not in ("s_branch", "s_endpgm", "s_setpc_b64") else [] for i in range(len(code))]
        for i, (name, ops) in enumerate(code):
            target = ops[0]
            if name == "s_setpc_b64":  # a far jump: its target stands in the sum before it
                target = re.search(r"\((\.\w+)-", code[i - 2][1][2])[1]
            if name.startswith(("s_branch", "s_cbranch", "s_setpc")) and labels[target] < len(code):
                before[labels[target]].append(i)

        def walk(i, reads, states):
            for p in before[i]:
                name, ops = code[p]
                if name.startswith("v_") and not name.startswith("v_mfma") and reads & _registers(ops[0]):
                    yield p
                passed = states + (int(ops[0], 0) + 1 if name == "s_nop" else 1)
                if passed < needed:
                    yield from walk(p, reads, passed)

        for i, (name, ops) in enumerate(code):
            if name.startswith("v_mfma"):
                reads = set().union(*(_registers(o) for o in ops[1:]))
                found += [(kernel, i, code[p], code[i]) for p in walk(i, reads, 0)]
    return found


SOURCES = ["mx.hip", "grouped_bf16.hip", "grouped_f16.hip"]


def _assembly(source):
    cmd = [build.hipcc(), *build.HIPCC_FLAGS, "-w", "--cuda-device-only", "-S", str(build.CSRC / source), "-o", "-"]
    return subprocess.run(cmd, capture_output=True, text=True)


@pytest.fixture(scope="module")
def assembly():
    with ThreadPoolExecutor(len(SOURCES)) as pool:  # a minute each
        return dict(zip(SOURCES, pool.map(_assembly, SOURCES)))


def test_the_check_sees_a_far_jump():
    code = "_Zk:\n.LBB0_1:\n\tv_mfma_f32_16x16x4_f32 a[0:3], v4, v5, a[0:3]\n\tv_lshrrev_b32_e32 v5, 8, v5\n{}"
    code += "\ts_add_u32 s54, s54, (.LBB0_1-.Lpost_getpc1)&4294967295\n\ts_addc_u32 s55, s55, (.LBB0_1-.Lpost_getpc1)>>32\n"
    code += "\ts_setpc_b64 s[54:55]\n.Lfunc_end0:\n"
    assert not hazards(code.format(""))  # the three scalar instructions are states enough
    assert len(hazards(code.format(""), 4)) == 1 and not hazards(code.format("\ts_nop 0\n"), 4)


def test_the_check_sees_a_missing_wait():
    code = "_Zk:\n\tv_mov_b32_e32 v5, v1\n{}\tv_mfma_f32_16x16x4_f32 a[0:3], v4, v[5:5], a[0:3]\n\ts_endpgm\n.Lfunc_end0:\n"
    assert len(hazards(code.format(""))) == 1
    assert len(hazards(code.format("\ts_nop 0\n"))) == 1
    assert not hazards(code.format("\ts_nop 1\n"))
    assert not hazards(code.format("\ts_nop 0\n\tds_read_b32 v6, v7\n"))
    assert not hazards(code.replace("v5, v1", "v6, v1").format(""))
    # around a loop: the write stands at the loop's end, the MFMA at its start
    loop = "_Zk:\n\ts_mov_b32 s0, 1\n.LBB0_1:\n\tv_mfma_f32_16x16x4_f32 a[0:3], v4, v5, a[0:3]\n\tv_lshrrev_b32_e32 v5, 8, v5\n"
    loop += "{}\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm\n.Lfunc_end0:\n"
    assert len(hazards(loop.format(""))) == 1 and not hazards(loop.format("\ts_nop 0\n"))


@pytest.mark.parametrize("source", SOURCES)
def test_wait_states_before_matrix_instructions(assembly, source):
    r = assembly[source]
    assert r.returncode == 0, r.stderr
    assert "v_mfma" in r.stdout
    assert not hazards(r.stdout)
