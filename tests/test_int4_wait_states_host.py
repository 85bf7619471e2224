"""The wait states before the matrix instructions of the 4-bit integer weights' kernels, whose bf16 operands come out of inline assembly: see
test_wait_states_host.py. Of each kernel the forms that differ in how codes become operands."""

import itertools
import subprocess

import pytest
from test_wait_states_host import hazards

from trnblas_amd import build

_FLAG = {False: "false", True: "true"}
FORMS = {
    "tile": ("int4_tile.hpp", [
        f"int4_tile_kernel<__bf16, {fm}, {fm}, {steps}, {_FLAG[zero]}, false, {_FLAG[gated]}>(GroupedArgs, Int4Args, int)"
        for fm, steps, zero, gated in [*itertools.product((4, 8), (1, 4), (False, True), (False,)), (4, 2, True, True), (8, 2, False, True)]
    ]),
    "rows": ("int4_rows.hpp", [
        f"int4_rows_kernel<__bf16, {p}, {mf}, {nf}, {steps}, {_FLAG[zero]}, {_FLAG[gated]}>(GroupedArgs, Int4Args, int)"
        for (p, mf, nf, gated), steps, zero in itertools.product([(1, 1, 1, False), (1, 4, 2, False), (3, 1, 2, True)], (1, 2, 4), (False, True))
    ]),
}  # fmt: skip


@pytest.mark.parametrize("kernel", list(FORMS))
def test_wait_states_before_matrix_instructions(tmp_path, kernel):
    header, forms = FORMS[kernel]
    lines = [f'#include "{build.CSRC / header}"', "namespace trnblas {", *(f"template __global__ void {f};" for f in forms), "}"]
    source = tmp_path / f"{kernel}.hip"
    source.write_text("\n".join(lines) + "\n")
    cmd = [build.hipcc(), *build.HIPCC_FLAGS, "-w", "--cuda-device-only", "-S", str(source), "-o", "-"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert r.stdout.count(".amdhsa_kernel ") == len(forms) and "v_mfma" in r.stdout and "v_cvt_off_f32_i4" in r.stdout
    assert not hazards(r.stdout)
