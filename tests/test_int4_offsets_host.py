"""The plan of gated products with 4-bit weights keeps to what the tile kernel reaches with 32-bit offsets: it reads the scales of gates and
ups from one buffer of 0x7ffffff0 bytes, N / 16 * ceil(K / 128) * (128 / steps) bytes apart, `steps` of 32 values to a group."""

import ctypes

import pytest

from trnblas_amd.hip import _lib

REACH = 0x7FFFFFF0
BF16, F16 = 1, 2


def plan(dtype, gated, groups, rows, N, K, group):
    out = (ctypes.c_int32 * 5)()
    _lib.call("trnblas_hip_int4_plan", dtype, gated, groups, rows, N, K, group, out)
    return list(out)


def last_inside(K, group):
    """The largest N, a multiple of 16, at which the ups' scales of a chunk lie within reach."""
    of_chunk = 128 * 32 // group  # bytes of a row block's scales of 128 values of K, which are read at once
    return (REACH - of_chunk) // (of_chunk * -(-K // 128)) * 16


# K: a multiple of 128 and not, one chunk, and small ones that a product of N and K says nothing about
@pytest.mark.parametrize("K", [1, 8, 100, 128, 129, 1024, 1032, 4096])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_tiles_stay_within_reach(K, group):
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    served = 0
    for dtype in (BF16, F16):
        for rows in (32, 64, 300, 2048):
            for N in (last_inside(K, group), last_inside(K, group) - 16 * 7):
                if N < 1 << 30:
                    served += plan(dtype, 1, 1, rows, N, K, group)[0] > 0
            for N in (last_inside(K, group) + 16, last_inside(K, group) + 16 * 9, 2 * last_inside(K, group), (1 << 30) - 2048):
                if last_inside(K, group) < N < 1 << 30:
                    assert plan(dtype, 1, 1, rows, N, K, group)[0] == 0, (rows, N)
    assert served or last_inside(K, group) >= 1 << 30 or K <= 128


@pytest.mark.parametrize("rows, N, K", [(32, 29826176, 1032), (2048, 1 << 28, 100), (2048, 1 << 27, 129)])
def test_sizes_past_reach(rows, N, K):
    # N K below 16 * 2^31, the offset at or past 2^31
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    assert plan(BF16, 1, 1, rows, N, K, 32)[0] == 0


def test_products_without_a_gate_keep_their_tiles():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    assert plan(BF16, 0, 1, 2048, 1 << 29, 100, 32)[0] > 0 and plan(BF16, 1, 1, 2048, 8192, 4096, 32)[0] > 0
