"""The wait states before the matrix instructions of the 4-bit integer weights' kernels, whose bf16 operands come out of inline assembly: see
test_wait_states_host.py."""

from concurrent.futures import ThreadPoolExecutor

import pytest
from test_wait_states_host import _assembly, hazards

SOURCES = ["int4_bf16.hip", "int4_tile_bf16.hip"]


@pytest.fixture(scope="module")
def assembly():
    with ThreadPoolExecutor(len(SOURCES)) as pool:  # up to two minutes each
        return dict(zip(SOURCES, pool.map(_assembly, SOURCES)))


@pytest.mark.parametrize("source", SOURCES)
def test_wait_states_before_matrix_instructions(assembly, source):
    r = assembly[source]
    assert r.returncode == 0, r.stderr
    assert "v_mfma" in r.stdout and not hazards(r.stdout)
