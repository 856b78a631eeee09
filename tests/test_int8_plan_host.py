"""Which kernel an 8-bit product takes, without a GPU (plans are those of 256 CUs there)."""

import ctypes

import pytest

from int8_helpers import CASES, plan

from bitnet_tt import _native as N


@pytest.fixture(scope="module")
def L():
    return N.lib()


@pytest.mark.parametrize("tile,shape,halves", CASES)
def test_the_tile_of_a_shape(L, tile, shape, halves):
    assert plan(L, *shape) == (0, *tile, halves)


@pytest.mark.parametrize("shape,blocks", [
    ((1, 16, 1), 1), ((32, 2560, 32768), 1), ((32, 2560, 32769), 2), ((33, 2560, 640), 0), ((16, 2576, 4096), 1),
    ((16, 2576, 4097), 0), ((17, 2576, 100), 0),
])
def test_few_rows_are_a_stream_of_weights(L, shape, blocks):
    assert plan(L, *shape)[0] == blocks


@pytest.mark.parametrize("shape", [(0, 64, 10), (4, 24, 10), (4, 16400, 10), (4, 64, 0), (-1, 64, 10), (4, 64, (1 << 24) + 1),
                                   (1 << 24, 64, 1 << 24)])
def test_plan_of_what_no_call_takes(L, shape):
    assert L.btl_int8_matmul_plan(*shape, (ctypes.c_int64 * 4)()) == 0
